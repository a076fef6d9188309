// Eviction from the paged cache by accumulated attention weight.
//
// Per (layer run, sequence, kv head) with L rows held and room for `keep`: the `recent` rows of highest position stay, and of the
// others the keep - recent of largest sum (ties: the lowest row). The kept rows at and behind `keep` move into the rows below it
// that are given up, the j-th kept into the j-th free one, so that rows 0 .. keep - 1 are the cache afterwards. Attention takes its
// keys in any order and keys are stored rotated, so a moved row is as good as before; its position moves with its sum. Sources lie
// at or behind `keep` and destinations below it: the rows move in place, in any order, and no more of them than have to.
//
// Two launches: a block per head finds what stays (the n-th largest key of 32 bits by its digits, eight bits a pass, then the rows in
// order), and blocks over all moves of all heads copy the rows.
#include "common.cuh"

namespace {

constexpr int MAX_SEQS = 128;  // sequences of a launch: their slots and lengths are arguments
struct Sequences {
  int slot[MAX_SEQS], length[MAX_SEQS];
};

constexpr int THREADS = 512, WARPS = THREADS / 32;

// Order of a sum as an unsigned number: a NaN counts as the largest, zeros are equal.
__device__ __forceinline__ unsigned order_of(float x) {
  const unsigned u = __float_as_uint(x == 0.f ? 0.f : x);
  return x != x ? 0xffffffffu : (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ unsigned order_of(int p) { return (unsigned)p ^ 0x80000000u; }

struct Line {
  unsigned value;
  int row;  // of the rows of exactly `value`, those up to this one are above the line
  __device__ __forceinline__ bool above(unsigned key, int r) const { return key > value || (key == value && r <= row); }
};

struct Scratch {
  int hist[256];
  int warp_sum[WARPS];
  unsigned value;
  int want, equal, row;
};

// Sum of `v` over the threads before this one (the block's total in `total`). All threads call it.
__device__ __forceinline__ int scan_before(int v, Scratch& sc, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) sc.warp_sum[warp] = x;
  __syncthreads();
  int before = 0;
  total = 0;
  for (int w = 0; w < WARPS; ++w) {
    if (w < warp) before += sc.warp_sum[w];
    total += sc.warp_sum[w];
  }
  return before + x - v;
}

// The line above which exactly n of the rows 0 .. L - 1 lie that `key` gives a value for (its second result).
template <typename Key>
__device__ Line line_of(int n, int L, Scratch& sc, Key key) {
  if (n <= 0) return Line{0xffffffffu, -1};
  unsigned prefix = 0, mask = 0;
  int want = n;
  for (int shift = 24; shift >= 0; shift -= 8) {
    __syncthreads();
    for (int i = threadIdx.x; i < 256; i += THREADS) sc.hist[i] = 0;
    __syncthreads();
    for (int r = threadIdx.x; r < L; r += THREADS) {
      unsigned v;
      if (key(r, v) && (v & mask) == prefix) atomicAdd(&sc.hist[(v >> shift) & 255], 1);
    }
    __syncthreads();
    if (threadIdx.x < 32) {  // lane: eight digits from the top
      int mine = 0;
      for (int i = 0; i < 8; ++i) mine += sc.hist[255 - (threadIdx.x * 8 + i)];
      int x = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if ((int)threadIdx.x >= o) x += y;
      }
      int above = x - mine;
      if (above < want && x >= want) {
        for (int i = 0; i < 8; ++i) {
          const int digit = 255 - (threadIdx.x * 8 + i), c = sc.hist[digit];
          if (above + c >= want) {
            sc.value = prefix | ((unsigned)digit << shift);
            sc.want = want - above;
            sc.equal = c;
            break;
          }
          above += c;
        }
      }
    }
    __syncthreads();
    prefix = sc.value;
    want = sc.want;
    mask |= 255u << shift;
  }
  Line line{prefix, 0x7fffffff};
  if (sc.equal > want) {  // more rows of this value than are wanted: the first of them
    if (threadIdx.x == 0) sc.row = -1;
    int seen = 0;
    for (int r0 = 0; r0 < L && seen < want; r0 += THREADS) {
      const int r = r0 + threadIdx.x;
      unsigned v;
      const bool is = r < L && key(r, v) && v == prefix;
      int total;
      const int before = seen + scan_before(is, sc, total);
      if (is && before == want - 1) sc.row = r;
      seen += total;
    }
    __syncthreads();
    line.row = sc.row;
  }
  return line;
}

__global__ void __launch_bounds__(THREADS)
choose_rows_kernel(const float* scores, const int* positions, float* scores_out, int* positions_out, size_t run_stride, int HKV, int capacity,
                   const Sequences seqs, int n_seqs, int keep, int recent, int* __restrict__ moves, int* __restrict__ n_moves, int max_moves,
                   int* seq_start, int* row_pos, int* seq_shift) {
  __shared__ Scratch sc;
  grid_launch_dependents();
  grid_dependency_wait();
  const int kh = blockIdx.x % HKV, seq = blockIdx.x / HKV % n_seqs, run = blockIdx.x / HKV / n_seqs;
  const int L = seqs.length[seq];
  const size_t base = run * run_stride + ((size_t)seqs.slot[seq] * HKV + kh) * capacity;
  const float* sum = scores + base;
  const int* pos = positions + base;
  float* sum_out = scores_out + base;
  int* pos_out = positions_out + base;
  const bool apart = sum != sum_out, pos_apart = pos != pos_out;
  if (L <= keep) {
    for (int r = threadIdx.x; r < L; r += THREADS) {
      if (apart) sum_out[r] = sum[r];
      if (pos_apart) pos_out[r] = pos[r];
    }
    if (threadIdx.x == 0) n_moves[blockIdx.x] = 0;
    return;
  }
  if (seq_start && kh == 0 && run == 0 && threadIdx.x == 0) {  // the step's description follows
    seq_start[seq] -= L - keep;
    row_pos[seq] -= L - keep;
    seq_shift[seq] += L - keep;
  }
  const Line newest = line_of(recent, L, sc, [&](int r, unsigned& v) { v = order_of(pos[r]); return true; });
  const Line heavy = line_of(keep - recent, L, sc, [&](int r, unsigned& v) {
    v = order_of(sum[r]);
    return !newest.above(order_of(pos[r]), r);
  });
  // the rows in order: free ones below `keep`, kept ones from there on
  int* to = moves + (size_t)blockIdx.x * 2 * max_moves;
  int* from = to + max_moves;
  int n_free = 0, n_kept = 0;
  for (int r0 = 0; r0 < L; r0 += THREADS) {
    const int r = r0 + threadIdx.x;
    bool kept = false;
    if (r < L) kept = newest.above(order_of(pos[r]), r) || heavy.above(order_of(sum[r]), r);
    const bool is_free = r < keep && !kept, moves_down = r >= keep && r < L && kept;
    // a chunk of rows may lie on both sides of `keep`: both counts in one scan
    int total;
    const int before = scan_before((is_free ? 1 : 0) | (moves_down ? 1 << 16 : 0), sc, total);
    if (is_free) to[n_free + (before & 0xffff)] = r;
    if (moves_down) from[n_kept + (before >> 16)] = r;
    if (r < keep && kept) {
      if (apart) sum_out[r] = sum[r];
      if (pos_apart) pos_out[r] = pos[r];
    }
    n_free += total & 0xffff;
    n_kept += total >> 16;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n_kept; i += THREADS) {
    const int s = from[i], d = to[i];
    sum_out[d] = sum[s];
    pos_out[d] = pos[s];
  }
  if (threadIdx.x == 0) n_moves[blockIdx.x] = n_kept;
}

// Piece: uint4, unsigned, unsigned short; a row is `pieces` of them.
constexpr int MOVE_THREADS = 256;
template <typename Piece>
__global__ void __launch_bounds__(MOVE_THREADS)
move_rows_kernel(Piece* k, Piece* v, size_t k_run, size_t v_run, int k_pieces, int v_pieces, int HKV, const Sequences seqs, int n_seqs,
                 const int* __restrict__ table, int width, const int* __restrict__ moves, const int* __restrict__ n_moves, int max_moves,
                 int blocks_per_head) {
  grid_launch_dependents();
  grid_dependency_wait();
  const int head = blockIdx.x / blocks_per_head, part = blockIdx.x % blocks_per_head;
  const int n = n_moves[head];
  const int kh = head % HKV, seq = head / HKV % n_seqs, run = head / HKV / n_seqs;
  const int* to = moves + (size_t)head * 2 * max_moves;
  const int* from = to + max_moves;
  const int* row = table + (size_t)seqs.slot[seq] * width;
  const int both = k_pieces + v_pieces;
  constexpr int AHEAD = 4;
  const long long total = (long long)n * both, step = (long long)blocks_per_head * MOVE_THREADS;
  for (long long i0 = (long long)part * MOVE_THREADS + threadIdx.x; i0 < total; i0 += step * AHEAD) {
    Piece got[AHEAD];
    Piece* dst[AHEAD];
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      const long long i = i0 + a * step;
      dst[a] = nullptr;
      if (i < total) {
        const int move = (int)(i / both), c = (int)(i % both), s = from[move], d = to[move];
        const bool key = c < k_pieces;
        Piece* pool = key ? k + run * k_run : v + run * v_run;
        const int pieces = key ? k_pieces : v_pieces, at = key ? c : c - k_pieces;
        got[a] = pool[(((size_t)row[s / KRK_PAGE] * HKV + kh) * KRK_PAGE + s % KRK_PAGE) * pieces + at];
        dst[a] = pool + (((size_t)row[d / KRK_PAGE] * HKV + kh) * KRK_PAGE + d % KRK_PAGE) * pieces + at;
      }
    }
#pragma unroll
    for (int a = 0; a < AHEAD; ++a)
      if (dst[a]) *dst[a] = got[a];
  }
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
  cudaError_t e = launch_pdl(choose_rows_kernel, dim3((unsigned)heads), dim3(THREADS), 0, stream, scores, positions, scores_out, positions_out,
                             (size_t)run_stride, HKV, capacity, seqs, n_seqs, keep, recent, moves, n_moves, max_moves, seq_start, row_pos, seq_shift);
  if (e != cudaSuccess) return (int)e;
  if (max_moves == 0) return 0;
  const long long align = k_row_bytes | (v ? v_row_bytes : 0) | k_run_bytes | (v ? v_run_bytes : 0) | (long long)(uintptr_t)k | (long long)(uintptr_t)v;
  auto go = [&](auto piece) {
    typedef decltype(piece) Piece;
    const int size = (int)sizeof(Piece), kp = k_row_bytes / size, vp = v ? v_row_bytes / size : 0;
    // enough blocks that a thread has one batch of pieces in flight, no more than fill the device a few times over
    const long long wanted = ((long long)max_moves * (kp + vp) + 4 * MOVE_THREADS - 1) / (4 * MOVE_THREADS);
    const long long room = (148 * 16 + heads - 1) / heads;
    const int per_head = (int)(wanted < room ? wanted : room);
    if (heads * per_head > 0x7fffffffLL) return -3;
    return (int)launch_pdl(move_rows_kernel<Piece>, dim3((unsigned)(heads * per_head)), dim3(MOVE_THREADS), 0, stream, (Piece*)k, (Piece*)v,
                           (size_t)(k_run_bytes / size), (size_t)(v_run_bytes / size), kp, vp, HKV, seqs, n_seqs, table, width, (const int*)moves,
                           (const int*)n_moves, max_moves, per_head);
  };
  if (align % 16 == 0) return go(uint4());
  if (align % 4 == 0) return go(0u);
  return go((unsigned short)0);
}
