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
  grid_launch_dependents();
  grid_dependency_wait();
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
// Every type, any size: t[r, p * wide + j] = scale sum_k x[r, k] A[a, p * rank + j, k] in 32 bits, a warp a sum
// ---------------------------------------------------------------------------------------------------------------------
//
// A sum's order depends on K alone, so a row gives the same bits whatever stands beside it.
template <typename T>
__global__ void __launch_bounds__(256) first_factor_kernel(float* __restrict__ t, const T* __restrict__ x, long long ldx, int K, const __grid_constant__ AdapterBank bank,
                                                           const int* __restrict__ row_adapter, int rows, int* __restrict__ error) {
  grid_launch_dependents();
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int per_row = bank.parts * bank.rank;
  for (int r = blockIdx.y; r < rows; r += gridDim.y) {
    const int a = row_adapter[r];
    if (a < 0 || a >= bank.capacity) {
      if (a >= bank.capacity && threadIdx.x == 0) atomicExch(error, KRK_ERROR_ADAPTER);
      continue;
    }
    for (int i = blockIdx.x * 8 + warp; i < per_row; i += gridDim.x * 8) {
      const int p = i / bank.rank, j = i % bank.rank;
      if (j >= bank.ranks[a * bank.parts + p]) continue;
      const T* w = reinterpret_cast<const T*>(bank.a) + ((size_t)a * per_row + i) * K;
      const T* xr = x + (size_t)r * ldx;
      float sum = 0.f;
      for (int k = lane; k < K; k += 32) sum += to_float<T>(xr[k]) * to_float<T>(w[k]);
      sum = warp_sum(sum);
      if (lane == 0) t[((size_t)r * bank.parts + p) * bank.wide + j] = sum * bank.scale[a * bank.parts + p];
    }
  }
}

// out[r, n] = y[r, n] + sum_j t[r, p of n, j] B[a, n, j], y in 32 bits, rounded once; gated: out = silu(gate) * up of the two halves.
template <typename T>
__device__ __forceinline__ float second_factor(const AdapterBank& bank, const float* t, int a, int r, int n, int N) {
  const int p = part_of(bank, n), rank = bank.ranks[a * bank.parts + p];
  const T* b = reinterpret_cast<const T*>(bank.b) + ((size_t)a * N + n) * bank.rank;
  const float* tr = t + ((size_t)r * bank.parts + p) * bank.wide;
  float sum = 0.f;
  for (int j = 0; j < rank; ++j) sum += tr[j] * to_float<T>(b[j]);
  return sum;
}

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
    float v = y[(size_t)r * N + n];
    if (a >= 0) v += second_factor<T>(bank, t, a, r, n, N);
    if (gated) {
      float u = y[(size_t)r * N + width + n];
      if (a >= 0) u += second_factor<T>(bank, t, a, r, width + n, N);
      v = v / (1.0f + expf(-v)) * u;
    }
    out[(size_t)r * width + n] = from_float<T>(v);
  }
}

}  // namespace

// The maps of a step of n_seqs sequences and n_rows rows. Optional: adapters, table (with slots and pages, of which n_pages are given). `words` takes, in order:
// with `places` row_place (two words a row); cu [n_seqs + 1], row_seq and row_pos [n_rows]; with adapters, on a boundary of two words each, row_adapter [n_rows], and for
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
    m.row_place = table ? reinterpret_cast<long long*>(words) : nullptr;
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

// t [rows, parts * wide] float32 of every row that has an adapter.
KRK_API int krk_adapter_first(float* t, const void* x, long long ldx, int rows, int K, const AdapterBank* bank, const int* row_adapter, int* error, int dtype,
                              cudaStream_t stream) {
  if (rows == 0) return 0;
  const dim3 grid((bank->parts * bank->rank + 7) / 8, min(rows, 32768));
  if (dtype == KRK_DTYPE_F32) return (int)launch_pdl(first_factor_kernel<float>, grid, dim3(256), 0, stream, t, (const float*)x, ldx, K, *bank, row_adapter, rows, error);
  if (dtype == KRK_DTYPE_BF16) return (int)launch_pdl(first_factor_kernel<bf16>, grid, dim3(256), 0, stream, t, (const bf16*)x, ldx, K, *bank, row_adapter, rows, error);
  return -4;
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
