"""What the cache's operators ask of their arguments before anything is launched (no GPU): pages, tables, slots and devices that a kernel would read or
write out of range."""

from types import SimpleNamespace

import pytest
import torch

from cache_ops_helpers import make_step
from kernel_rush_kawk_b200.csrc import cache_ops
from kernel_rush_kawk_b200.csrc.cache_ops import CacheOps, KernelError


class Checks(CacheOps):
    error = torch.zeros(1, dtype=torch.int32)


@pytest.fixture(autouse=True)
def a_device(monkeypatch):
    monkeypatch.setattr(cache_ops, "_current_device", lambda: -1)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: -1)


def step():
    return make_step("cpu", torch.bfloat16, 4, 2, 32, [70, 80], [1, 1], 1, ([2], [64]))


def check(qkv, batch, cache):
    return Checks()._check_step("attention", qkv, 4, 2, 32, batch, cache)


def elsewhere(t):
    """A tensor like this one on another device."""
    return type("Elsewhere", (), dict(get_device=lambda self: 1, device="cuda:1", __getattr__=lambda self, name: getattr(t, name)))()


def test_a_step_that_fits_is_taken():
    qkv, batch, cache = step()
    assert check(qkv, batch, cache) == (qkv.data_ptr(), qkv.stride(0), cache.k.data_ptr(), cache.v.data_ptr())


@pytest.mark.parametrize("change", [
    dict(v=lambda c: c.v[:-1]), dict(k=lambda c: c.k[:-1]), dict(k=lambda c: c.k.view(c.k.shape[0], 1, 128, 32)),
    dict(k=lambda c: c.k.view(-1, 2, 32, 32), v=lambda c: c.v.view(-1, 2, 32, 32)), dict(v=lambda c: c.v.float()), dict(table=lambda c: c.table.long()),
    dict(table=lambda c: c.table[:, :-1]), dict(table=lambda c: c.table.t().contiguous().t()), dict(table=lambda c: c.table[:, :-1].contiguous()),
    dict(table=lambda c: c.table[:2].contiguous()), dict(v=lambda c: elsewhere(c.v)), dict(table=lambda c: elsewhere(c.table)), dict(k=lambda c: elsewhere(c.k))])
def test_caches_that_do_not_fit(change):
    qkv, batch, cache = step()
    batch.slots[0] = 3
    changed = SimpleNamespace(**{**vars(cache), **{name: f(cache) for name, f in change.items()}})
    with pytest.raises(KernelError):
        check(qkv, batch, changed)


def test_steps_that_do_not_fit():
    qkv, batch, cache = step()
    for slots in ([0, 4], [-1, 0]):
        with pytest.raises(KernelError, match="slots"):
            check(qkv, SimpleNamespace(**{**vars(batch), "slots": slots}), cache)
    with pytest.raises(KernelError, match="cuda:1"):
        check(qkv, SimpleNamespace(**{**vars(batch), "cu_q": elsewhere(batch.cu_q)}), cache)


def test_evictions_that_do_not_fit():
    k = torch.zeros((2, 5, 1, 64, 8))
    table, counts = torch.zeros((3, 2), dtype=torch.int32), (2, 3, 1, 128)
    scores, positions = torch.zeros(counts), torch.zeros(counts, dtype=torch.int32)

    def evict(k=k, v=k.clone(), table=table, batch=None):
        Checks().evict_keys(k, v, table, [0], [100], scores, positions, 10, 3, batch=batch)

    step = lambda **kw: SimpleNamespace(**{**dict(n_seqs=1, n_rows=1, seq_start=scores, seq_shift=scores), **kw})
    for kw in [dict(k=k[:1].expand(2, -1, -1, -1, -1)), dict(v=k[:1].expand(2, -1, -1, -1, -1)), dict(table=table.view(-1)), dict(table=table.float()),
               dict(batch=step(seq_shift=elsewhere(scores))), dict(batch=step(seq_start=elsewhere(scores))), dict(batch=step(n_rows=2)), dict(v=elsewhere(k)), dict(table=elsewhere(table))]:
        with pytest.raises(KernelError):
            evict(**kw)


def test_a_slot_whose_sums_two_sequences_would_add_to():
    qkv, batch, cache = step()
    batch.slots = [1, 1]
    with pytest.raises(KernelError, match="every slot comes once"):
        Checks().scored_attention(qkv, 4, 2, 32, batch, cache, 0.1, torch.zeros((cache.table.shape[0], 2, cache.width * 64)))
