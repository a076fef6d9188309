// Who multiplies what of a product with adapters (adapted_gemm.cu): tiles, and shares of tiles. Plain arithmetic, for the host and the device.
#pragma once

namespace {

constexpr int PAIRS = 74;  // of SMs

// The most pairs that bring a share of one of `rest` tiles.
__host__ inline int shares_of_a_tile(int rest) { return (PAIRS + rest - 1) / rest + 1; }
// As many pairs a tile, where that leaves few of them idle: fewer shares, and no pair has two. Else 0.
__host__ inline int aligned_parts(int rest, int k_blocks) {
  const int each = PAIRS / rest;
  return rest * each * 10 >= PAIRS * 9 ? (each < k_blocks ? each : k_blocks) : 0;
}

// The work of a pair: of the tiles before `shared`, tiles pair, pair + pairs, ... as a whole; of the tiles from there on a share. A tile has its blocks of k
// and, where there is a single row tile, its adapters (else they go to who `ends` its k). With `aligned` a tile is dealt to so many pairs, blocks and
// adapters in equal parts; else the blocks and adapters of all tiles, in order, to all pairs, `run` from pair * run on.
struct Walk {
  int k_blocks, extra, shared, run, aligned, at, end, whole, pairs;
  __host__ __device__ Walk(int pair, int pairs_, int tiles, int shared_, int k_blocks_, int extra_, int aligned_)
      : k_blocks(k_blocks_), extra(extra_), shared(shared_), aligned(aligned_), whole(pair), pairs(pairs_) {
    const int units = k_blocks + extra, all = units * (tiles - shared);
    if (aligned) {  // tile and part
      run = 1;
      at = min(pair, (tiles - shared) * aligned);
      end = min(pair + 1, (tiles - shared) * aligned);
    } else {
      run = max(1, (int)(((long long)all + pairs - 1) / pairs));
      at = (int)min((long long)pair * run, (long long)all);
      end = (int)min((long long)at + run, (long long)all);
    }
  }
  // tile t, of which blocks of k from k0 to k1, adapters from e0 to e1
  __host__ __device__ bool next(int& t, int& k0, int& k1, int& e0, int& e1) {
    if (whole < shared) {
      t = whole;
      whole += pairs;
      k0 = e0 = 0;
      k1 = k_blocks;
      e1 = extra;
      return true;
    }
    if (at >= end) return false;
    if (aligned) {
      const int part = at % aligned, ks = (k_blocks + aligned - 1) / aligned, es = (extra + aligned - 1) / aligned;
      t = shared + at / aligned;
      k0 = min(k_blocks, part * ks);
      k1 = min(k_blocks, k0 + ks);
      e0 = min(extra, part * es);
      e1 = min(extra, e0 + es);
      at = end;
      return true;
    }
    // from behind: a run begins with what it has of its last tile, whose t it does not need, and waits for t where nothing is left to load but that
    const int units = k_blocks + extra, of = (end - 1) / units, u1 = end - of * units, u0 = max(0, at - of * units);
    t = shared + of;
    k0 = min(k_blocks, u0);
    k1 = min(k_blocks, u1);
    e0 = max(0, u0 - k_blocks);
    e1 = max(0, u1 - k_blocks);
    end -= u1 - u0;
    return true;
  }
  // Whether a part has the last block of k. (Of 217 blocks in 24 parts of ten the last two have none, and end nothing.)
  __host__ __device__ bool ends(int k0, int k1) const { return k0 < k1 && k1 == k_blocks; }
  __host__ __device__ int first_pair(int t) const { return aligned ? (t - shared) * aligned : (int)((long long)(t - shared) * (k_blocks + extra) / run); }
  __host__ __device__ int count(int t) const { return aligned ? aligned : (int)(((long long)(t - shared + 1) * (k_blocks + extra) - 1) / run) - first_pair(t) + 1; }
};

}  // namespace
