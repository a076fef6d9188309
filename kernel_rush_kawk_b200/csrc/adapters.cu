// The maps of a step, from its requests' lengths, and the adapters' products for every type: the first factor's rows, and the second
// factor's added to what the shared projection gave.
#include "adapters.cuh"
#include "mma.cuh"

namespace {

// ---------------------------------------------------------------------------------------------------------------------
// Maps of a step
// ---------------------------------------------------------------------------------------------------------------------
//
// One launch, whose blocks do not wait on one another: each adds up all sequences' lengths and new pages for itself (a thousand sequences
// are 8 KB out of L2) and takes 768 rows, which are whole tiles of 128, 192 and 256. A row finds its sequence by bisection. The row at the
// first position of a new page writes the table's entry; places of other rows on that page come from the list of pages, not from the table.
// A tile's slots begin at (tile + sequence of its first row): every earlier tile had no more adapters than sequences, and a sequence is
// counted once more for each tile that it goes on into, so tiles never meet in them, and no block needs another's count.
//
// Its bytes are next to nothing (40,432 rows of 16 prompts: 0.8 MB): latency bounds it. Replayed: 64 single tokens 4.6 us, these prompts 8.3, 120,600 rows of a thousand
// sequences 15.1 (two passes over all lengths in every block, then the tiles' adapters, a warp a tile). One call 17.3 to 18.1 us of the host's
// time, of which the launch 4, the buffer 2.5, the views 5.
constexpr int MAP_ROWS = 768, MAP_THREADS = 256;

struct Maps {
  const int *slots, *starts, *lengths, *adapters;
  int n_seqs, n_rows;
  int* table;
  int width, n_slots;
  const int* pages;
  int n_pages;
  int *cu, *row_seq, *row_pos, *row_adapter;
  long long* row_place;
  int* info[3];
  int* list[3];
  int tile_rows[3];
  int n_lists;
  int* error;
};

__device__ __forceinline__ int pages_of(long long positions) { return (int)((positions + KRK_PAGE - 1) / KRK_PAGE); }

__global__ void __launch_bounds__(MAP_THREADS) step_maps_kernel(const Maps m) {
  extern __shared__ int seq_maps[];
  int* cu = seq_maps;                   // [n_seqs + 1] first rows
  int* fresh = seq_maps + m.n_seqs + 1;  // [n_seqs + 1] first of the new pages
  __shared__ long long warp_rows[MAP_THREADS / 32], warp_pages[MAP_THREADS / 32];
  __shared__ int found[MAP_THREADS / 32][256];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  grid_dependency_wait();  // (and no later kernel is let in: some read a step's description and page table before they wait for the one before)
  // lengths and new pages of all sequences, added up: a thread's run of sequences, the threads' sums, the runs again
  const int each = (m.n_seqs + MAP_THREADS - 1) / MAP_THREADS, s0 = min(tid * each, m.n_seqs), s1 = min(s0 + each, m.n_seqs);
  long long rows = 0, pages = 0;
  bool bad = false;
  auto length_of = [&](int s) {
    const int n = m.lengths[s];
    if (n < 0 || n > m.n_rows) bad = true;
    return min(max(n, 0), m.n_rows);
  };
  auto start_of = [&](int s) {
    const int n = m.starts[s];
    if (n < 0) bad = true;
    return max(n, 0);
  };
  for (int s = s0; s < s1; ++s) {
    const int n = length_of(s), start = start_of(s);
    rows += n;
    pages += pages_of((long long)start + n) - pages_of(start);
  }
  long long upto_rows = rows, upto_pages = pages;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long a = __shfl_up_sync(0xffffffffu, upto_rows, o), b = __shfl_up_sync(0xffffffffu, upto_pages, o);
    if (lane >= o) {
      upto_rows += a;
      upto_pages += b;
    }
  }
  if (lane == 31) {
    warp_rows[warp] = upto_rows;
    warp_pages[warp] = upto_pages;
  }
  __syncthreads();
  long long row = upto_rows - rows, page = upto_pages - pages;
  for (int w = 0; w < warp; ++w) {
    row += warp_rows[w];
    page += warp_pages[w];
  }
  for (int s = s0; s < s1; ++s) {
    cu[s] = (int)min(row, (long long)m.n_rows);
    fresh[s] = (int)min(page, (long long)INT_MAX);
    const int n = length_of(s), start = start_of(s);
    row += n;
    page += pages_of((long long)start + n) - pages_of(start);
  }
  if (tid == MAP_THREADS - 1) {
    bad |= row != m.n_rows;
    cu[m.n_seqs] = (int)min(row, (long long)m.n_rows);
    fresh[m.n_seqs] = (int)min(page, (long long)INT_MAX);
    if (m.table) bad |= page > m.n_pages;
  }
  __syncthreads();
  if (blockIdx.x == 0)
    for (int s = tid; s <= m.n_seqs; s += MAP_THREADS) m.cu[s] = cu[s];

  const int covered = cu[m.n_seqs];
  // the last sequence whose first row is no later than r, which has rows since r is one of them
  auto seq_of = [&](int r) {
    int lo = 0, hi = m.n_seqs;  // cu[lo] <= r < cu[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (cu[mid] <= r) lo = mid; else hi = mid;
    }
    return lo;
  };
  const int first = blockIdx.x * MAP_ROWS, last = min(first + MAP_ROWS, m.n_rows);
  for (int r = first + tid; r < last; r += MAP_THREADS) {
    int seq = 0, adapter = -1;
    long long pos = -1, place = -1;
    if (r < covered) {
      seq = seq_of(r);
      const int start = max(m.starts[seq], 0);
      pos = (long long)start + (r - cu[seq]);
      if (m.adapters) adapter = m.adapters[seq];
      if (m.table) {
        const int slot = m.slots[seq], have = pages_of(start);
        const long long b = pos / KRK_PAGE;
        if ((unsigned)slot >= (unsigned)m.n_slots || b >= m.width) {
          bad = true;
        } else {
          int* entry = m.table + (size_t)slot * m.width + b;
          int at;
          if (b < have) {
            at = *entry;
            bad |= at < 0;
          } else {
            const long long i = fresh[seq] + (b - have);
            at = i < m.n_pages ? m.pages[i] : -1;
            if (at < 0) bad = true;
            else if (pos % KRK_PAGE == 0) *entry = at;
          }
          if (at >= 0) place = (long long)at * KRK_PAGE + pos % KRK_PAGE;
        }
      }
      if (pos > INT_MAX) {
        bad = true;
        pos = -1;
      }
    }
    m.row_seq[r] = seq;
    m.row_pos[r] = (int)pos;
    if (m.row_place) m.row_place[r] = place;
    if (m.row_adapter) m.row_adapter[r] = adapter;
  }
  if (bad) atomicExch(m.error, KRK_ERROR_MAPS);

  // the adapters of every tile that begins in this block's rows, a warp a tile
  for (int l = 0; l < m.n_lists; ++l) {
    const int tile_rows = m.tile_rows[l];
    for (int r0 = first + warp * tile_rows; r0 < last; r0 += MAP_THREADS / 32 * tile_rows) {
      const int tile = r0 / tile_rows;
      const int tiles = (m.n_rows + tile_rows - 1) / tile_rows;
      // where the slots of a tile begin: the first tile's at 0; behind the last sequence, as if there were one more
      auto begin_of = [&](int i) { return i == 0 ? 0 : i == tiles ? tiles + m.n_seqs : i + (i * tile_rows < covered ? seq_of(i * tile_rows) : m.n_seqs); };
      const int begin = begin_of(tile), end = begin_of(tile + 1);
      int count = 0;
      if (r0 < covered) {
        const int lo = seq_of(r0);
        const int hi = seq_of(min(min(r0 + tile_rows, m.n_rows), covered) - 1);
        for (int s = lo; s <= hi; s += 32) {
          const int mine = s + lane;
          const int a = mine <= hi && cu[mine + 1] > cu[mine] ? m.adapters[mine] : -1;
          bool is_new = a >= 0;
          for (int i = 0; i < count && is_new; ++i) is_new = found[warp][i] != a;
          const unsigned same = __match_any_sync(0xffffffffu, a);
          is_new = is_new && (__ffs(same) - 1) == lane;
          const unsigned all = __ballot_sync(0xffffffffu, is_new);
          const int at = count + __popc(all & ((1u << lane) - 1));
          if (is_new) {
            found[warp][at] = a;
            *reinterpret_cast<int2*>(m.list[l] + 2 * (begin + at)) = make_int2(a, tile);
          }
          count += __popc(all);
          __syncwarp();
        }
      }
      if (lane == 0) *reinterpret_cast<int2*>(m.info[l] + 2 * tile) = make_int2(begin, count);
      for (int i = begin + count + lane; i < end; i += 32) *reinterpret_cast<int2*>(m.list[l] + 2 * i) = make_int2(-1, tile);
      __syncwarp();
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// Every type, any size: t[r, p * wide + j] = scale sum_k x[r, k] A[a, p * rank + j, k] in 32 bits
// ---------------------------------------------------------------------------------------------------------------------
//
// A block has four columns of t and the rows, of sixteen neighbours, that have one adapter: A's rows are read once for four of them. Its eight warps take pieces of
// 128 k in turn, a lane four of a piece, whether or not addresses let it read them at once; lanes are added up, then warps in order. A sum's order so depends
// on K alone, and a row gives the same bits whatever stands beside it. Bound by the way to L2 of A, of whose rows a warp has a few in flight. (A warp a sum over
// all of K: sixteen rows, rank 64, K = 9,728: 130 us, and the product behind it waited.) Columns behind an adapter's rank, up to the next multiple of 16 of the
// bank's, are zeros.
constexpr int FIRST_COLS = 4, FIRST_WINDOW = 16;

template <typename T, bool WIDE>
__device__ __forceinline__ void four_of(float (&v)[4], const T* p, int n) {
  if constexpr (WIDE && sizeof(T) == 4) {
    const float4 all = *reinterpret_cast<const float4*>(p);
    v[0] = all.x; v[1] = all.y; v[2] = all.z; v[3] = all.w;
  } else if constexpr (WIDE) {
    const uint2 all = *reinterpret_cast<const uint2*>(p);
    v[0] = __uint_as_float(all.x << 16); v[1] = __uint_as_float(all.x & 0xffff0000u);
    v[2] = __uint_as_float(all.y << 16); v[3] = __uint_as_float(all.y & 0xffff0000u);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < n ? to_float<T>(p[i]) : 0.f;
  }
}

// R rows of one adapter; w: the first of the columns' rows of A
template <typename T, bool WIDE, int R>
__device__ __forceinline__ void first_sums(float* sums, const T* const (&x)[R], const T* w, int cols, int K, int lane, int warp) {
  float sum[R][FIRST_COLS];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int c = 0; c < FIRST_COLS; ++c) sum[r][c] = 0.f;
#pragma unroll 2
  for (int k = 128 * warp + 4 * lane; k < K; k += 128 * 8) {
    float u[R][4], v[FIRST_COLS][4];
#pragma unroll
    for (int c = 0; c < FIRST_COLS; ++c) four_of<T, WIDE>(v[c], w + (size_t)min(c, cols - 1) * K + k, K - k);
#pragma unroll
    for (int r = 0; r < R; ++r) four_of<T, WIDE>(u[r], x[r] + k, K - k);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int c = 0; c < FIRST_COLS; ++c) sum[r][c] = fmaf(u[r][i], v[c][i], sum[r][c]);
  }
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int c = 0; c < FIRST_COLS; ++c) {
      const float all = warp_sum(sum[r][c]);
      if (lane == 0) sums[(r * FIRST_COLS + c) * 8 + warp] = all;
    }
}

template <typename T, bool WIDE>
__global__ void __launch_bounds__(256) first_factor_kernel(float* __restrict__ t, const T* __restrict__ x, long long ldx, int K, const __grid_constant__ AdapterBank bank,
                                                           const int* __restrict__ row_adapter, int rows, int early, int* __restrict__ error) {
  __shared__ float sums[4 * FIRST_COLS * 8];
  grid_dependency_wait();
  if (early) grid_launch_dependents();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int column = blockIdx.x * FIRST_COLS, p = column / bank.wide, j = column % bank.wide;  // (wide is a multiple of 16)
  for (int r0 = blockIdx.y * FIRST_WINDOW; r0 < rows; r0 += gridDim.y * FIRST_WINDOW) {
    const int r = r0 + blockIdx.z;
    const int theirs = lane < FIRST_WINDOW && r0 + lane < rows ? row_adapter[r0 + lane] : -1;
    const int a = __shfl_sync(0xffffffffu, theirs, blockIdx.z);
    unsigned left = __ballot_sync(0xffffffffu, theirs == a);
    const int before = __popc(left & ((1u << blockIdx.z) - 1));
    if (r >= rows || a < 0 || before % 4) continue;  // (a row before this one has the adapter and takes this one along)
    if (a >= bank.capacity) {
      if (tid == 0) atomicExch(error, KRK_ERROR_ADAPTER);
      continue;
    }
    left &= ~((1u << blockIdx.z) - 1);
    const int cols = min(bank.ranks[a * bank.parts + p] - j, FIRST_COLS), n = min(__popc(left), 4);
    const float scale = bank.scale[a * bank.parts + p];
    const T* w = reinterpret_cast<const T*>(bank.a) + ((size_t)(a * bank.parts + p) * bank.rank + j) * K;
    {
      int at[4];
      const T* from[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        at[i] = r0 + (left ? __ffs(left) - 1 : blockIdx.z);
        left &= left - 1;
        from[i] = x + (size_t)at[i] * ldx;
      }
      if (cols > 0) {
        if (n == 1) {
          const T* const one[1] = {from[0]};
          first_sums<T, WIDE, 1>(sums, one, w, cols, K, lane, warp);
        } else if (n == 2) {
          const T* const two[2] = {from[0], from[1]};
          first_sums<T, WIDE, 2>(sums, two, w, cols, K, lane, warp);
        } else {
          const T* const four[4] = {from[0], from[1], from[2], from[3]};
          first_sums<T, WIDE, 4>(sums, four, w, cols, K, lane, warp);
        }
      }
      __syncthreads();
      grid_launch_dependents();
      if (tid < n * FIRST_COLS) {
        const int i = tid / FIRST_COLS, c = tid % FIRST_COLS;
        float all = 0.f;
        if (c < cols) {
#pragma unroll
          for (int s = 0; s < 8; ++s) all += sums[tid * 8 + s];
          all *= scale;
        }
        t[(size_t)at[i] * bank.parts * bank.wide + column + c] = all;
      }
      __syncthreads();
    }
  }
}

// out[r, n] = y[r, n] + sum_j t[r, p of n, j] B[a, n, j], y in 32 bits, rounded once; gated: out = silu(gate) * up of the two halves.
template <typename T>
__global__ void __launch_bounds__(256) second_factor_kernel(T* __restrict__ out, const float* __restrict__ y, const float* __restrict__ t, const __grid_constant__ AdapterBank bank,
                                                            const int* __restrict__ row_adapter, int rows, int N, int gated) {
  grid_launch_dependents();
  grid_dependency_wait();
  const int width = gated ? N / 2 : N;
  const int n = blockIdx.x * 256 + threadIdx.x;
  if (n >= width) return;
  for (int r = blockIdx.y; r < rows; r += gridDim.y) {
    int a = row_adapter[r];
    if (a >= bank.capacity) a = -1;
    const int whose[1] = {a}, row[1] = {r};
    float v;
    if (gated) {
      float sums[1][2] = {{y[(size_t)r * N + n], y[(size_t)r * N + width + n]}};
      const int at[2] = {n, width + n};
      add_second_factor<T, 1, 2>(bank, t, whose, row, at, sums);
      v = sums[0][0] / (1.0f + expf(-sums[0][0])) * sums[0][1];
    } else {
      float sums[1][1] = {{y[(size_t)r * N + n]}};
      const int at[1] = {n};
      add_second_factor<T, 1, 1>(bank, t, whose, row, at, sums);
      v = sums[0][0];
    }
    out[(size_t)r * width + n] = from_float<T>(v);
  }
}

}  // namespace

// The maps of a step of n_seqs sequences and n_rows rows. Optional: adapters, table (with slots and pages, of which n_pages are given). `words` takes, in order:
// with `places` row_place (two words a row, -1 without a table); cu [n_seqs + 1], row_seq and row_pos [n_rows]; with adapters, on a boundary of two words each, row_adapter [n_rows], and for
// tiles of 128, 192 and 256 rows, or of all rows up to a multiple of 32 where there are no more than 256, a tile's first slot and number of adapters, and the
// slots, one for each tile and sequence: an adapter and its tile.
KRK_API int krk_step_maps(const int* slots, const int* starts, const int* lengths, const int* adapters, int n_seqs, int n_rows, int* table, int width, int n_slots,
                          const int* pages, int n_pages, int* words, int places, int* error, cudaStream_t stream) {
  constexpr size_t MOST = 200 * 1024;
  const size_t smem = (size_t)(n_seqs + 1) * 8;
  if (n_seqs < 0 || n_rows < 0 || smem > MOST || ((uintptr_t)words & 7) || (table && !places)) return -2;
  Maps m = {slots, starts, lengths, adapters, n_seqs, n_rows, table, width, n_slots, pages, n_pages};
  int* const first = words;
  if (places) {
    m.row_place = reinterpret_cast<long long*>(words);
    words += 2 * (size_t)n_rows;
  }
  m.cu = words;
  m.row_seq = m.cu + n_seqs + 1;
  m.row_pos = m.row_seq + n_rows;
  words = m.row_pos + n_rows;
  if (adapters) {
    words += (words - first) & 1;
    m.row_adapter = words;
    words += n_rows + (n_rows & 1);
    const int all[3] = {128, 192, 256}, one = n_rows > 32 ? (n_rows + 31) / 32 * 32 : 32;
    m.n_lists = n_rows > 256 ? 3 : 1;
    for (int i = 0; i < m.n_lists; ++i) {
      const int height = m.n_lists == 1 ? one : all[i];
      const size_t tiles = ((size_t)n_rows + height - 1) / height;
      m.tile_rows[i] = height;
      m.info[i] = words;
      m.list[i] = words + 2 * tiles;
      words += 2 * (2 * tiles + n_seqs);
    }
  }
  m.error = error;
  static unsigned long long allowed = 0;
  if (smem > 32 * 1024) {
    const cudaError_t e = allow_shared(step_maps_kernel, MOST, &allowed);
    if (e != cudaSuccess) return (int)e;
  }
  const int blocks = n_rows > MAP_ROWS ? (n_rows + MAP_ROWS - 1) / MAP_ROWS : 1;
  return (int)launch_pdl(step_maps_kernel, dim3(blocks), dim3(MAP_THREADS), smem, stream, m);
}

int krk_first_factor_f32(float* t, const void* x, long long ldx, int rows, int K, const AdapterBank& bank, const int* row_adapter, int* error, int dtype,
                         cudaStream_t stream) {
  const dim3 grid(bank.parts * bank.wide / FIRST_COLS, min((rows + FIRST_WINDOW - 1) / FIRST_WINDOW, 32768), min(rows, FIRST_WINDOW));
  const bool wide = !((K | ldx) & 3) && !(((uintptr_t)x | (uintptr_t)bank.a) & 15);
  // The next kernel's blocks go to the SMs that have none of these first, and many of them on few SMs cost more than what they would stream beside these (eight rows of
  // K = 9,728, rank 64, 128 blocks here: 82 us and 63 behind them; four rows, 64 blocks: 47 and 51).
  const int early = (long long)grid.x * grid.y * grid.z <= 74;
  auto launch = [&](auto kernel, auto* typed) {
    return (int)launch_pdl(kernel, grid, dim3(256), 0, stream, t, typed, ldx, K, bank, row_adapter, rows, early, error);
  };
  if (dtype == KRK_DTYPE_F32) return launch(wide ? first_factor_kernel<float, true> : first_factor_kernel<float, false>, (const float*)x);
  if (dtype == KRK_DTYPE_BF16) return launch(wide ? first_factor_kernel<bf16, true> : first_factor_kernel<bf16, false>, (const bf16*)x);
  return -4;
}

// t [rows, parts * wide] float32 of every row that has an adapter.
KRK_API int krk_adapter_first(float* t, const void* x, long long ldx, int rows, int K, const AdapterBank* bank, const int* row_adapter, int* error, int dtype,
                              cudaStream_t stream) {
  return rows == 0 ? 0 : krk_first_factor_f32(t, x, ldx, rows, K, *bank, row_adapter, error, dtype, stream);
}

// out [rows, N] (gated: [rows, N / 2]) from y [rows, N] float32 and t.
KRK_API int krk_adapter_second(void* out, const float* y, const float* t, int rows, int N, const AdapterBank* bank, const int* row_adapter, int gated, int dtype,
                               cudaStream_t stream) {
  if (rows == 0 || N == 0) return 0;
  const dim3 grid(((gated ? N / 2 : N) + 255) / 256, min(rows, 32768));
  if (dtype == KRK_DTYPE_F32) return (int)launch_pdl(second_factor_kernel<float>, grid, dim3(256), 0, stream, (float*)out, y, t, *bank, row_adapter, rows, N, gated);
  if (dtype == KRK_DTYPE_BF16) return (int)launch_pdl(second_factor_kernel<bf16>, grid, dim3(256), 0, stream, (bf16*)out, y, t, *bank, row_adapter, rows, N, gated);
  return -4;
}
