"""Attention over shared prefixes right behind the maps that say where its sequences' rows begin: as with maps made long before."""

import pytest
import torch

from cache_ops_helpers import exact_attention, make_step
from kernel_rush_kawk_b200.cache.prefix import PrefixGroups, longer_steps_share
from kernel_rush_kawk_b200.csrc import load_kernels
from kernel_rush_kawk_b200.csrc.adapter_ops import StepMaps

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops():
    return load_kernels(())


@pytest.fixture(autouse=True)
def always_shared(monkeypatch):
    """Small cases take the kernels that large ones do."""
    from kernel_rush_kawk_b200.cache import prefix

    monkeypatch.setattr(prefix, "SHARE_BYTES", 0)
    monkeypatch.setattr(prefix, "JOIN_STEPS", -1e9)


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("heads,kv,dim,sizes,lengths,tokens", [
    (32, 8, 128, [8], [1024], 2),      # one tile
    (16, 2, 64, [4, 4], [2048, 2048], 2),
    (32, 8, 128, [16], [2048], 31),    # many
    (32, 8, 128, [32], [1024], 8)])
def test_right_behind_the_maps(ops, heads, kv, dim, sizes, lengths, tokens, captured):
    n, per = sum(sizes), heads // kv
    held = [length + (7 * i) % 50 for i, length in enumerate(length for size, length in zip(sizes, lengths) for _ in range(size))]
    brings = [tokens + i % 2 for i in range(n)]
    qkv, batch, cache = make_step(DEV, torch.bfloat16, heads, kv, dim, held, brings, seed=3, groups=(sizes, lengths))
    prefix = PrefixGroups(sizes, lengths, DEV)
    assert longer_steps_share(prefix.sizes, prefix.lengths, batch.q_lens, per, kv) and prefix.max_rows(batch) * per >= ops.PREFIX_TENSOR_ROWS
    attend = lambda: ops.shared_prefix_attention(qkv, heads, kv, dim, batch, cache, dim ** -0.5, prefix)
    want, off, _, _ = exact_attention(qkv, heads, kv, dim, batch, cache, dim ** -0.5)
    expected = attend()
    assert ((expected.double() - want).abs() <= off).all()
    maps = StepMaps(batch.n_rows, n, DEV, with_places=False, with_adapters=False)
    batch.cu_q, batch.row_seq, batch.row_pos = maps.cu_q, maps.row_seq, maps.row_pos

    def step():
        maps.buffer.zero_()  # no rows at all, for who reads too early
        ops.step_maps(batch.seq_slot, batch.seq_start, batch.seq_qlen, batch.n_rows, out=maps)
        return attend()

    if captured:
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = step()
    busy = torch.randn((8192, 8192), device=DEV, dtype=torch.bfloat16)
    for _ in range(10):
        busy @ busy  # what follows is queued behind it, all at once
        if captured:
            y.zero_()
            graph.replay()
        else:
            y = step()
        assert torch.equal(y, expected)
    ops.check()


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n", [1, 5, 64])
def test_single_tokens_right_behind_the_maps(ops, n, dim, captured):
    """Attention of tokens whose pages the maps have just entered."""
    heads, kv = 8, 2
    held = [64 * (i % 5) if i % 2 == 0 else 17 * i % 300 for i in range(n)]
    qkv, batch, cache = make_step(DEV, torch.bfloat16, heads, kv, dim, held, [1] * n, seed=4)
    cache.k.nan_to_num_(0)
    cache.v.nan_to_num_(0)
    wanted = cache.table.clone()
    table, k, v = cache.table, cache.k.clone(), cache.v.clone()
    fresh = [(s, h // 64) for s, h in zip(batch.slots, held) if h % 64 == 0]
    pages = torch.tensor([int(wanted[at]) for at in fresh], dtype=torch.int32, device=DEV)
    stale = wanted.clone()
    for at in fresh:
        stale[at] = 0  # some page, for who reads too early
    attend = lambda: ops.rope_attention(qkv, heads, kv, dim, None, None, 1e-6, None, None, batch, cache, dim ** -0.5, None)
    expected = attend().clone()
    after = cache.k.clone(), cache.v.clone()
    maps = StepMaps(n, n, DEV, with_adapters=False)

    def step():
        ops.step_maps(batch.seq_slot, batch.seq_start, batch.seq_qlen, n, table=table, pages=pages, out=maps)
        return attend()

    def before():
        table.copy_(stale)
        cache.k.copy_(k)
        cache.v.copy_(v)

    if captured:
        before()
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = step()
    busy = torch.randn((8192, 8192), device=DEV, dtype=torch.bfloat16)
    for _ in range(10):
        before()
        busy @ busy
        if captured:
            graph.replay()
        else:
            y = step()
        assert torch.equal(y, expected) and torch.equal(table, wanted)
        assert torch.equal(cache.k, after[0]) and torch.equal(cache.v, after[1])
    ops.check()
