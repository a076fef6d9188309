// Eviction from the paged cache by accumulated attention weight.
//
// Per (layer run, sequence, kv head) with L rows held and room for `keep`: the `recent` rows of highest position stay, and of the
// others the keep - recent of largest sum (ties: the lowest row). The kept rows at and behind `keep` move into the rows below it
// that are given up, the j-th kept into the j-th free one, so that rows 0 .. keep - 1 are the cache afterwards. Attention takes its
// keys in any order and keys are stored rotated, so a moved row is as good as before; its position moves with its sum. Sources lie
// at or behind `keep` and destinations below it: the rows move in place, in any order, and no more of them than have to.
//
// A block per head finds what stays: a line through the positions and one through the other rows' sums, then the rows in order. It moves the
// rows as well where there are heads enough; else blocks over all moves of all heads do, in a second launch.
//
// What bounds it is the finding: passes of one block over a head's rows in shared memory, with barriers between. The lines by bins of the numbers'
// range (two passes mostly) instead of a bisection of their bits: 58.8 to 26 us. 16 sequences of 1,088 rows to 1,024, 8 layers of 8 heads
// of 128 (1,024 heads, 82 MB): 27 us, of which the bytes would take 12.5. One prompt of 16,300 rows to 2,048 (64 heads, 129 MB): 22 us for the lines and
// 27 for the moves.
#include "common.cuh"

namespace {

constexpr int MAX_SEQS = 128;  // sequences of a launch: their slots and lengths are arguments
struct Sequences {
  int slot[MAX_SEQS], length[MAX_SEQS];
};

// Order of a sum as an unsigned number: a NaN counts as the largest, zeros are equal.
__device__ __forceinline__ unsigned order_of(float x) {
  const unsigned u = __float_as_uint(x == 0.f ? 0.f : x);
  return x != x ? 0xffffffffu : (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ unsigned order_of(int p) { return (unsigned)p ^ 0x80000000u; }

// Lists of a block of T threads; behind it, in dynamic shared memory, the rows' keys (STAGED) and a bit for each row that is kept.
constexpr int MAX_CANDIDATES = 512, FEW = 64;
template <int T, int BINS>
struct Scratch {
  static constexpr int COPIES = T > 128 ? 4 : 1;
  int hist[BINS * COPIES];  // counters of a bin side by side, a lane's by its number: many rows of one warp fall into the same bins
  unsigned cand_key[MAX_CANDIDATES];
  int cand_row[MAX_CANDIDATES];
  int part[2][32];
  unsigned low, high;
  int bin, want, n_cand, row;
};

// A line through the rows' keys: exactly the wanted number of rows lies above it.
struct Line {
  unsigned value;
  int row;  // of the rows of exactly `value`, those up to this one
  __device__ __forceinline__ bool above(unsigned key, int r) const { return key > value || (key == value && r <= row); }
};

// The block's least and largest of the threads' (lo, hi).
template <int T, int BINS>
__device__ __forceinline__ void block_range(unsigned& lo, unsigned& hi, Scratch<T, BINS>& sc) {
  lo = __reduce_min_sync(0xffffffffu, lo);
  hi = __reduce_max_sync(0xffffffffu, hi);
  if (threadIdx.x == 0) { sc.low = 0xffffffffu; sc.high = 0; }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) { atomicMin(&sc.low, lo); atomicMax(&sc.high, hi); }
  __syncthreads();
  lo = sc.low;
  hi = sc.high;
}

// The line above which exactly n of the rows 0 .. L - 1 lie that `key` gives a value for (its second result), all of them from lo to hi; n
// is at most their number. The range is cut into bins; the one that the line falls into holds few rows mostly, whose order is
// counted out pair by pair, else it is the next range.
// DENSE: numbers of which the n largest may be neighbours (positions), which one count shows.
template <bool DENSE, int T, int BINS, typename Key>
__device__ Line line_of(int n, int L, unsigned lo, unsigned hi, Scratch<T, BINS>& sc, Key key) {
  if (n <= 0) return Line{0xffffffffu, -1};
  constexpr int BITS = BINS == 512 ? 9 : 11, EACH = BINS / T, COPIES = Scratch<T, BINS>::COPIES;
  static_assert(1 << BITS == BINS && BINS % T == 0, "");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (DENSE && hi - lo >= (unsigned)n) {
    int mine = 0;
#pragma unroll 4
    for (int r = threadIdx.x; r < L; r += T) {
      unsigned v;
      mine += key(r, v) && v > hi - n;
    }
    mine = __reduce_add_sync(0xffffffffu, mine);
    if (lane == 0) sc.part[0][warp] = mine;
    __syncthreads();
    const int count = __reduce_add_sync(0xffffffffu, lane < T / 32 ? sc.part[0][lane] : 0);
    if (count == n) return Line{hi - n + 1, 0x7fffffff};
  }
  int want = n;
  for (;;) {
    const int shift = max(0, 32 - __clz(hi - lo) - BITS);  // (a range of one value: shift 0)
#pragma unroll
    for (int i = 0; i < EACH * COPIES; ++i) sc.hist[threadIdx.x + i * T] = 0;
    if (threadIdx.x == 0) sc.n_cand = 0;
    __syncthreads();
#pragma unroll 4
    for (int r = threadIdx.x; r < L; r += T) {
      unsigned v;
      if (key(r, v) && v - lo <= hi - lo) atomicAdd(&sc.hist[((v - lo) >> shift) * COPIES + lane % COPIES], 1);
    }
    __syncthreads();
    auto count_of = [&](int bin) {
      int c = 0;
#pragma unroll
      for (int e = 0; e < COPIES; ++e) c += sc.hist[bin * COPIES + e];
      return c;
    };
    int mine = 0;  // of a thread's bins, from the top
#pragma unroll
    for (int i = 0; i < EACH; ++i) mine += count_of(BINS - 1 - (threadIdx.x * EACH + i));
    int x = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) sc.part[1][warp] = x;
    __syncthreads();
    int above = x - mine + __reduce_add_sync(0xffffffffu, lane < warp ? sc.part[1][lane] : 0);
    if (above < want && above + mine >= want)
      for (int i = 0; i < EACH; ++i) {
        const int at = BINS - 1 - (threadIdx.x * EACH + i), c = count_of(at);
        if (above + c >= want) {
          sc.bin = at;
          sc.want = want - above;
          break;
        }
        above += c;
      }
    __syncthreads();
    const int in_bin = count_of(sc.bin);
    lo += (unsigned)sc.bin << shift;
    hi = lo + min(hi - lo, (1u << shift) - 1);
    want = sc.want;
    if (in_bin == want) return Line{lo, 0x7fffffff};  // the bin as a whole (a key on its lower edge counts with all of its rows)
    if (in_bin <= FEW || (shift == 0 && in_bin <= MAX_CANDIDATES)) {  // (of more, another cut leaves fewer, and costs less than their pairs)
#pragma unroll 4
      for (int r = threadIdx.x; r < L; r += T) {
        unsigned v;
        if (key(r, v) && v - lo <= hi - lo) {
          const int c = atomicAdd(&sc.n_cand, 1);
          sc.cand_key[c] = v;
          sc.cand_row[c] = r;
        }
      }
      __syncthreads();
      for (int c = threadIdx.x; c < in_bin; c += T) {
        const unsigned v = sc.cand_key[c];
        const int r = sc.cand_row[c];
        int before = 0;
#pragma unroll 8
        for (int e = 0; e < in_bin; ++e) before += sc.cand_key[e] > v || (sc.cand_key[e] == v && sc.cand_row[e] < r);
        if (before == want - 1) { sc.low = v; sc.row = r; }
      }
      __syncthreads();
      return Line{sc.low, sc.row};
    }
    if (shift == 0) break;  // more rows of one value than the list holds
    __syncthreads();        // the table is cleared for the next range
  }
  // the first of the rows of this value
  if (threadIdx.x == 0) sc.row = -1;
  int seen = 0;
  for (int r0 = 0; r0 < L && seen < want; r0 += T) {
    const int r = r0 + threadIdx.x;
    unsigned v;
    const bool is = r < L && key(r, v) && v == lo;
    const unsigned votes = __ballot_sync(0xffffffffu, is);
    __syncthreads();
    if (lane == 0) sc.part[0][warp] = __popc(votes);
    __syncthreads();
    const int here = lane < T / 32 ? sc.part[0][lane] : 0;
    const int before = seen + __reduce_add_sync(0xffffffffu, lane < warp ? here : 0) + __popc(votes & ((1u << lane) - 1));
    if (is && before == want - 1) sc.row = r;
    seen += __reduce_add_sync(0xffffffffu, here);
  }
  __syncthreads();
  return Line{lo, sc.row};
}

struct Pools {  // of keys and of values, as pieces of 16, 4 or 2 bytes; a row is `pieces` of them
  void *k, *v;
  size_t k_run, v_run;  // between runs, in pieces
  int k_pieces, v_pieces;
  const int* table;
  int width, piece_bytes;
};

// Rows `from` to rows `to` of one head, this thread's share of n moves: `workers` threads share them, 32 or fewer lanes a move.
template <typename Piece>
__device__ __forceinline__ void move_rows(const Pools& p, const int* __restrict__ to, const int* __restrict__ from, int n, int run, int slot, int kh, int HKV,
                                          int worker, int workers) {
  const int both = p.k_pieces + p.v_pieces;
  int lanes = 32;  // of a warp that share a move
  while (lanes > 1 && lanes >= 2 * both) lanes >>= 1;
  const int first = worker / lanes, step = workers / lanes, c0 = worker % lanes;
  const int* row = p.table + (size_t)slot * p.width;
  Piece* kp = reinterpret_cast<Piece*>(p.k) + run * p.k_run;
  Piece* vp = reinterpret_cast<Piece*>(p.v) + run * p.v_run;
  constexpr int AHEAD = 4;  // moves whose rows are on their way together
  for (int m0 = first; m0 < n; m0 += step * AHEAD) {
    int s[AHEAD], d[AHEAD];
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      const int m = m0 + a * step;
      s[a] = m < n ? from[m] : -1;
      d[a] = m < n ? to[m] : 0;
    }
    size_t sr[AHEAD], dr[AHEAD];
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      sr[a] = s[a] < 0 ? 0 : ((size_t)row[s[a] / KRK_PAGE] * HKV + kh) * KRK_PAGE + s[a] % KRK_PAGE;
      dr[a] = s[a] < 0 ? 0 : ((size_t)row[d[a] / KRK_PAGE] * HKV + kh) * KRK_PAGE + d[a] % KRK_PAGE;
    }
    for (int c = c0; c < both; c += lanes) {
      const bool key = c < p.k_pieces;
      Piece* pool = key ? kp : vp;
      const int pieces = key ? p.k_pieces : p.v_pieces, at = key ? c : c - p.k_pieces;
      Piece got[AHEAD];
#pragma unroll
      for (int a = 0; a < AHEAD; ++a)
        if (s[a] >= 0) got[a] = pool[sr[a] * pieces + at];
#pragma unroll
      for (int a = 0; a < AHEAD; ++a)
        if (s[a] >= 0) pool[dr[a] * pieces + at] = got[a];
    }
  }
}

__device__ __forceinline__ void move_rows(const Pools& p, const int* to, const int* from, int n, int run, int slot, int kh, int HKV, int worker, int workers) {
  if (p.piece_bytes == 16) move_rows<uint4>(p, to, from, n, run, slot, kh, HKV, worker, workers);
  else if (p.piece_bytes == 4) move_rows<unsigned>(p, to, from, n, run, slot, kh, HKV, worker, workers);
  else move_rows<unsigned short>(p, to, from, n, run, slot, kh, HKV, worker, workers);
}

struct ChooseArgs {
  const float* scores;
  const int* positions;
  float* scores_out;
  int* positions_out;
  size_t run_stride;
  int HKV, capacity, n_seqs, keep, recent, max_moves;
  int *moves, *n_moves;
  int *seq_start, *row_pos, *seq_shift;
  bool move_here;
};

// A block for a head: what stays, the moves, and, where there are heads enough to fill the device, the moving. STAGED: the rows' keys lie in
// shared memory, each read once from the cache's tables; else every reading goes to memory again.
template <int T, int BINS, bool STAGED>
__global__ void __launch_bounds__(T)
choose_rows_kernel(const ChooseArgs a, const Sequences seqs, const Pools pools, int staged_rows) {
  __shared__ Scratch<T, BINS> sc;
  extern __shared__ __align__(16) unsigned dynamic_s[];
  unsigned *pos_s = dynamic_s, *sum_s = dynamic_s + staged_rows;  // order_of each; a sum that does not stand for election becomes 0, which no number has
  unsigned* kept_s = dynamic_s + 2 * staged_rows;
  grid_dependency_wait();
  if (!a.seq_start) grid_launch_dependents();  // kernels read a step's description before they wait for the one before: none overtakes its change
  const int kh = blockIdx.x % a.HKV, seq = blockIdx.x / a.HKV % a.n_seqs, run = blockIdx.x / a.HKV / a.n_seqs;
  const int L = seqs.length[seq], keep = a.keep;
  const size_t base = run * a.run_stride + ((size_t)seqs.slot[seq] * a.HKV + kh) * a.capacity;
  const float* sum = a.scores + base;
  const int* pos = a.positions + base;
  float* sum_out = a.scores_out + base;
  int* pos_out = a.positions_out + base;
  const bool apart = sum != sum_out, pos_apart = pos != pos_out;
  if (L <= keep) {
    for (int r = threadIdx.x; r < L; r += T) {
      if (apart) sum_out[r] = sum[r];
      if (pos_apart) pos_out[r] = pos[r];
    }
    if (threadIdx.x == 0) a.n_moves[blockIdx.x] = 0;
    return;
  }
  if (a.seq_start && kh == 0 && run == 0 && threadIdx.x == 0) {  // the step's description follows
    a.seq_start[seq] -= L - keep;
    a.row_pos[seq] -= L - keep;
    a.seq_shift[seq] += L - keep;
  }
  unsigned lo = 0xffffffffu, hi = 0;
  constexpr int READS = 8;  // rows of a thread that are on their way together
  for (int r0 = threadIdx.x; r0 < L; r0 += T * READS) {
    int p[READS];
    float x[READS];
#pragma unroll
    for (int e = 0; e < READS; ++e) {
      const int r = min(r0 + e * T, L - 1);
      p[e] = pos[r];
      x[e] = STAGED ? sum[r] : 0.f;
    }
#pragma unroll
    for (int e = 0; e < READS; ++e) {
      const int r = min(r0 + e * T, L - 1);  // (the last row more than once)
      const unsigned v = order_of(p[e]);
      if (STAGED) {
        pos_s[r] = v;
        sum_s[r] = order_of(x[e]);
      }
      lo = min(lo, v);
      hi = max(hi, v);
    }
  }
  block_range(lo, hi, sc);
  const Line newest = line_of<true>(a.recent, L, lo, hi, sc, [&](int r, unsigned& v) { v = STAGED ? pos_s[r] : order_of(pos[r]); return true; });
  auto key = [&](int r, unsigned& v) {
    if (STAGED) {
      v = sum_s[r];
      return v != 0;
    }
    v = order_of(sum[r]);
    return !newest.above(order_of(pos[r]), r);
  };
  lo = 0xffffffffu;
  hi = 0;
#pragma unroll 4
  for (int r = threadIdx.x; r < L; r += T) {
    unsigned v;
    if (STAGED && newest.above(pos_s[r], r)) sum_s[r] = 0;
    if (key(r, v)) { lo = min(lo, v); hi = max(hi, v); }
  }
  __syncthreads();
  block_range(lo, hi, sc);
  const Line heavy = line_of<false>(keep - a.recent, L, lo, hi, sc, key);
  // the rows' bits; how many are free below `keep`, and kept from there on, in each warp's share of the words
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr int WARPS = T / 32;
  const int words = (L + 31) / 32, per = (words + WARPS - 1) / WARPS, w_lo = warp * per, w_hi = min(words, w_lo + per);
  int n_free = 0, n_down = 0;
  for (int w = w_lo; w < w_hi; ++w) {
    const int r = 32 * w + lane;
    unsigned v;
    const bool stays = r < L && (!key(r, v) || heavy.above(v, r));
    const unsigned bits = __ballot_sync(0xffffffffu, stays), below = __ballot_sync(0xffffffffu, r < keep);
    if (lane == 0) kept_s[w] = bits;
    n_free += __popc(~bits & below);
    n_down += __popc(bits & ~below);
  }
  __syncthreads();
  if (lane == 0) { sc.part[0][warp] = n_free; sc.part[1][warp] = n_down; }
  __syncthreads();
  int at_free = __reduce_add_sync(0xffffffffu, lane < warp ? sc.part[0][lane] : 0);
  int at_down = __reduce_add_sync(0xffffffffu, lane < warp ? sc.part[1][lane] : 0);
  const int n_moves = __reduce_add_sync(0xffffffffu, lane < WARPS ? sc.part[1][lane] : 0);
  int* to = a.moves + (size_t)blockIdx.x * 2 * a.max_moves;
  int* from = to + a.max_moves;
  for (int w = w_lo; w < w_hi; ++w) {
    const int r = 32 * w + lane;
    const unsigned bits = kept_s[w], below = __ballot_sync(0xffffffffu, r < keep), before = (1u << lane) - 1;
    if ((~bits & below) >> lane & 1) to[at_free + __popc(~bits & below & before)] = r;
    if ((bits & ~below) >> lane & 1) from[at_down + __popc(bits & ~below & before)] = r;
    at_free += __popc(~bits & below);
    at_down += __popc(bits & ~below);
  }
  __syncthreads();
  constexpr int AHEAD = 4;  // rows of a thread that are on their way together
  if (apart || pos_apart)
    for (int r0 = threadIdx.x; r0 < keep; r0 += T * AHEAD) {
      float x[AHEAD];
      int p[AHEAD];
      bool stays[AHEAD];
#pragma unroll
      for (int e = 0; e < AHEAD; ++e) {
        const int r = r0 + e * T;
        stays[e] = r < keep && (kept_s[r / 32] >> (r % 32) & 1);
        if (stays[e]) { x[e] = sum[r]; p[e] = pos[r]; }
      }
#pragma unroll
      for (int e = 0; e < AHEAD; ++e)
        if (stays[e]) {
          if (apart) sum_out[r0 + e * T] = x[e];
          if (pos_apart) pos_out[r0 + e * T] = p[e];
        }
    }
  for (int i0 = threadIdx.x; i0 < n_moves; i0 += T * AHEAD) {
    int s[AHEAD], d[AHEAD], p[AHEAD];
    float x[AHEAD];
#pragma unroll
    for (int e = 0; e < AHEAD; ++e) {
      const int i = i0 + e * T;
      s[e] = i < n_moves ? from[i] : -1;
      d[e] = i < n_moves ? to[i] : 0;
    }
#pragma unroll
    for (int e = 0; e < AHEAD; ++e)
      if (s[e] >= 0) { x[e] = sum[s[e]]; p[e] = pos[s[e]]; }
#pragma unroll
    for (int e = 0; e < AHEAD; ++e)
      if (s[e] >= 0) { sum_out[d[e]] = x[e]; pos_out[d[e]] = p[e]; }
  }
  if (a.move_here) move_rows(pools, to, from, n_moves, run, seqs.slot[seq], kh, a.HKV, threadIdx.x, T);
  else if (threadIdx.x == 0) a.n_moves[blockIdx.x] = n_moves;
}

constexpr int MOVE_THREADS = 256;
__global__ void __launch_bounds__(MOVE_THREADS)
move_rows_kernel(const Pools pools, int HKV, const Sequences seqs, int n_seqs, const int* __restrict__ moves, const int* __restrict__ n_moves, int max_moves,
                 int blocks_per_head) {
  grid_dependency_wait();
  grid_launch_dependents();
  const int head = blockIdx.x / blocks_per_head, part = blockIdx.x % blocks_per_head;
  const int kh = head % HKV, seq = head / HKV % n_seqs, run = head / HKV / n_seqs;
  const int* to = moves + (size_t)head * 2 * max_moves;
  move_rows(pools, to, to + max_moves, n_moves[head], run, seqs.slot[seq], kh, HKV, part * MOVE_THREADS + threadIdx.x, blocks_per_head * MOVE_THREADS);
}

}  // namespace

KRK_API int krk_evict_max_seqs(void) { return MAX_SEQS; }

// slots, lengths: host arrays of n_seqs <= MAX_SEQS. moves: [runs * n_seqs * HKV][2][max_moves] and n_moves [runs * n_seqs * HKV] are scratch; max_moves
// at least min(keep, longest - keep). Row bytes: of one position of one kv head. v null: keys serve as values. Strides between runs in bytes
// (pools) and elements (scores). seq_start, row_pos, seq_shift: the description of a step of these sequences, or null.
KRK_API int krk_evict_keys(void* k, void* v, long long k_run_bytes, long long v_run_bytes, int k_row_bytes, int v_row_bytes, int HKV, int runs,
                           const int* table, int width, const float* scores, const int* positions, float* scores_out, int* positions_out,
                           long long run_stride, int capacity, const int* slots, const int* lengths, int n_seqs, int keep, int recent, int* moves,
                           int* n_moves, int max_moves, int* seq_start, int* row_pos, int* seq_shift, cudaStream_t stream) {
  if (n_seqs == 0 || runs == 0) return 0;
  if (n_seqs > MAX_SEQS || keep < 1 || recent < 0 || recent > keep) return -2;
  const long long heads = (long long)runs * n_seqs * HKV;
  if (heads > 0x7fffffffLL) return -3;
  Sequences seqs = {};
  for (int i = 0; i < n_seqs; ++i) { seqs.slot[i] = slots[i]; seqs.length[i] = lengths[i]; }
  const long long align = k_row_bytes | (v ? v_row_bytes : 0) | k_run_bytes | (v ? v_run_bytes : 0) | (long long)(uintptr_t)k | (long long)(uintptr_t)v;
  const int piece = align % 16 == 0 ? 16 : align % 4 == 0 ? 4 : 2;
  const Pools pools = {k, v, (size_t)(k_run_bytes / piece), (size_t)(v_run_bytes / piece), k_row_bytes / piece, v ? v_row_bytes / piece : 0, table, width, piece};
  // A head's block moves its rows itself where there are two heads an SM or more, or little to move.
  const bool move_here = heads >= 296 || (long long)max_moves * (k_row_bytes + v_row_bytes) <= 32768;
  const ChooseArgs args = {scores, positions, scores_out, positions_out, (size_t)run_stride, HKV, capacity, n_seqs, keep, recent, max_moves,
                           moves, n_moves, seq_start, row_pos, seq_shift, move_here};
  int longest = 0;
  for (int i = 0; i < n_seqs; ++i) longest = lengths[i] > longest ? lengths[i] : longest;
  // Few rows: few threads, whose sums and barriers cost more than the rows do. Many rows of few heads: as many threads as a block has (64 heads of 16,300 rows
  // 58.4 us by 512 threads and 54.3 by 1,024, 128 of 8,000 54.3 and 50.2; 256 of 8,000 85.0 and 89.1). Rows whose keys do not fit shared memory are
  // read again.
  static unsigned long long allowed[4] = {0, 0, 0, 0};
  constexpr size_t MOST = 190 * 1024;
  auto choose = [&](auto* kern, int threads, int staged) {
    const size_t smem = (size_t)staged * 8 + ((size_t)longest + 31) / 32 * 4;
    const cudaError_t e = smem > MOST ? cudaErrorInvalidValue : allow_shared(kern, MOST, allowed + (threads > 128) + (threads > 512) + (threads > 512 && staged));
    return e != cudaSuccess ? e : launch_pdl(kern, dim3((unsigned)heads), dim3(threads), smem, stream, args, seqs, pools, staged);
  };
  cudaError_t e = longest <= 2048    ? choose(choose_rows_kernel<128, 512, true>, 128, longest)
                  : heads <= 148 && longest > 6000 && longest <= 23000 ? choose(choose_rows_kernel<1024, 2048, true>, 1024, longest)
                  : longest <= 23000 ? choose(choose_rows_kernel<512, 2048, true>, 512, longest)
                                     : choose(choose_rows_kernel<1024, 2048, false>, 1024, 0);
  if (e != cudaSuccess || max_moves == 0 || move_here) return (int)e;
  // four moves in flight a warp's share, and no more blocks than fill the device a few times over
  const long long wanted = ((long long)max_moves * 32 + 4 * MOVE_THREADS - 1) / (4 * MOVE_THREADS), room = (148 * 8 + heads - 1) / heads;
  const int per_head = (int)(wanted < room ? wanted : room);
  if (heads * per_head > 0x7fffffffLL) return -3;
  return (int)launch_pdl(move_rows_kernel, dim3((unsigned)(heads * per_head)), dim3(MOVE_THREADS), 0, stream, pools, HKV, seqs, n_seqs, (const int*)moves,
                         (const int*)n_moves, max_moves, per_head);
}
