// pages.cu -- block tables and slot maps from the lengths of the requests.
#include "tkb_common.cuh"
#include "../../include/tkm_b200.h"

namespace tkb {

// Latency bounds it: some 20 bytes a sequence and 8 a page moved.  One launch
// of one cluster (one CTA for small calls): every CTA sums the sequences'
// needs for itself (a scan over at most 4096 of them, in shared memory), so
// that the CTAs share nothing but the order of three phases, kept by cluster
// barriers: all have read the state; surplus pages are on the stack; the
// missing ones are in the table.  The slots of many rows are a second launch
// over all SMs (1000 sequences, 190 k rows: 84 us in the cluster's eight).
struct PagesParams {
  int32_t* table;
  int32_t* held;
  const int32_t* lens;
  int32_t* free_pages;
  int32_t* n_free;
  int32_t* granted;
  long long* slots;
  const int32_t* row_start;
  int rows;  // without slots: about how many tokens come and go
  int B, max_pages, page_size, n_pages;
};

// Exclusive sums over the block of each thread's value, and the total.
template <int THREADS, typename V>
TKB_DEVFN V block_scan(V v, V* s_warp, V& total) {
  constexpr int W = THREADS / 32;
  const int lane = lane_id(), w = warp_id();
  V x = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const V y = __shfl_up_sync(0xffffffffu, x, d);
    if (lane >= d) x += y;
  }
  __syncthreads();
  if (lane == 31) s_warp[w] = x;
  __syncthreads();
  const V sum = lane < W ? s_warp[lane] : V(0);
  V upto = sum;
#pragma unroll
  for (int d = 1; d < W; d <<= 1) {
    const V y = __shfl_up_sync(0xffffffffu, upto, d);
    if (lane >= d) upto += y;
  }
  total = __shfl_sync(0xffffffffu, upto, W - 1);
  const V before = __shfl_sync(0xffffffffu, upto - sum, w);
  return before + x - v;
}

// Whether a number names a page; the error bit where it does not.
TKB_DEVFN bool page_ok(const PagesParams& p, int page) {
  if (static_cast<unsigned>(page) < static_cast<unsigned>(p.n_pages)) return true;
  atomicOr(&g_device_error, ERR_BAD_INDEX);
  return false;
}
// The slot of a row that belongs to sequence b, `back` rows before its sequence's end.
TKB_DEVFN long long page_slot(const PagesParams& p, int b, int back, int pages) {
  const long long slot = static_cast<long long>(__ldg(p.lens + b)) - back;
  if (slot < 0 || slot >= static_cast<long long>(pages) * p.page_size) return -1;
  const int i = static_cast<int>(slot) / p.page_size;
  const int page = __ldcg(p.table + static_cast<long long>(b) * p.max_pages + i);
  if (!page_ok(p, page)) return -1;
  return static_cast<long long>(page) * p.page_size + (static_cast<int>(slot) - i * p.page_size);
}
// The sequence of a row: the last b with row_start[b] <= row; false where the row is not its own.
TKB_DEVFN bool row_seq(const int32_t* row_start, int B, int row, int& b, int& back) {
  b = row;
  back = 1;
  if (!row_start) return true;
  int lo = 0, hi = B - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (__ldg(row_start + mid) <= row) lo = mid;
    else hi = mid - 1;
  }
  b = lo;
  const int end = __ldg(row_start + b + 1);
  back = end - row;
  return __ldg(row_start + b) <= row && row < end;
}

// One CTA of 256 threads or the cluster, us a call in a graph without slots, B sequences of which each moves so many pages:
//   B          16            32            48            64            96            128           256
//   none   1.8   4.1     2.1   4.2     2.5   4.3     2.8   4.2     3.3   4.2     3.9   4.2     6.3   4.2
//   8      2.3   4.5     3.0   4.6     3.7   4.6     4.5   4.6     6.0   4.8     7.4   4.5    13.6   4.5
//   128    3.4   5.1     5.2   5.2     7.0   5.3     8.8   5.3    12.7   5.3    16.2   5.2    30.8   5.3
//   512    8.0   7.4    14.2   7.9    20.7   7.9    26.5   8.0    39.1   8.1    51.4   7.9     101   8.1
// Up to kPagesFew rows are steps, which move next to nothing.  More are prompts, and of those the slots are a second launch
// (64 sequences, 10 k rows: in one CTA 18 us, in the cluster 12.3, apart 11.1).
constexpr int kPagesFew = 1024;
static bool pages_one_cta(const PagesParams& p) {
  return p.rows <= kPagesFew ? p.B <= 128 : p.B <= 48 && p.rows / p.page_size <= 4096;
}

// SEQS sequences a thread.
template <int THREADS, int SEQS>
__global__ void __launch_bounds__(THREADS) kv_pages_kernel(const __grid_constant__ PagesParams p) {
  // per sequence: pages kept, pages to give back (with a minus sign) or to take, and where they go on or come off the stack
  extern __shared__ int s_seq[];
  __shared__ unsigned long long s_warp[32];
  int* s_kept = s_seq;
  int* s_move = s_seq + p.B;
  int* s_at = s_seq + 2 * p.B;
  const int tid = threadIdx.x, lane = lane_id();
  const int rank = blockIdx.x, ctas = gridDim.x;  // the grid is one cluster
  auto together = [&]() {
    if (SEQS > 1) cluster_sync();
    else __syncthreads();
  };
  grid_wait();
  int kept[SEQS], back[SEQS], need[SEQS], sum_back = 0, sum_need = 0;
  bool odd = false, room[SEQS];
  const long long most = static_cast<long long>(p.max_pages) * p.page_size;
#pragma unroll
  for (int i = 0; i < SEQS; ++i) {
    const int b = tid * SEQS + i;
    kept[i] = back[i] = need[i] = 0;
    room[i] = true;
    if (b >= p.B) continue;
    int held = p.held[b], n = p.lens[b];
    odd |= held < 0 || held > p.max_pages || n < 0;
    held = min(max(held, 0), p.max_pages);
    n = max(n, 0);
    room[i] = n <= most;
    const int want = static_cast<int>(min(static_cast<long long>(p.max_pages), (n + static_cast<long long>(p.page_size) - 1) / p.page_size));
    kept[i] = min(held, want);
    back[i] = held - kept[i];
    need[i] = want - kept[i];
    sum_back += back[i];
    sum_need += need[i];
  }
  int n_free = *p.n_free;
  odd |= n_free < 0 || n_free > p.n_pages;
  n_free = min(max(n_free, 0), p.n_pages);
  unsigned long long all;
  const unsigned long long at = block_scan<THREADS>(static_cast<unsigned long long>(sum_back) << 32 | static_cast<unsigned>(sum_need), s_warp, all);
  const int all_back = static_cast<int>(all >> 32);
  int at_back = n_free + static_cast<int>(at >> 32), at_need = static_cast<int>(at & 0xffffffffu);
  odd |= n_free + all_back > p.n_pages;
  const int height = min(n_free + all_back, p.n_pages);
  together();  // all have read held and n_free
  int taken = 0;
#pragma unroll
  for (int i = 0; i < SEQS; ++i) {
    const int b = tid * SEQS + i;
    if (b >= p.B) break;
    const bool fits = need[i] == 0 || at_need + need[i] <= height;
    s_kept[b] = kept[i];
    s_move[b] = back[i] ? -back[i] : fits ? need[i] : 0;
    s_at[b] = back[i] ? at_back : height - 1 - at_need;
    if (rank == 0) {
      p.held[b] = kept[i] + (fits ? need[i] : 0);
      if (p.granted) p.granted[b] = fits && room[i];
    }
    at_back += back[i];
    at_need += need[i];
    if (fits && need[i]) taken = at_need;
  }
  taken = __reduce_max_sync(0xffffffffu, taken);
  __syncthreads();
  if (lane == 0) s_warp[warp_id()] = static_cast<unsigned>(taken);
  __syncthreads();
  if (tid == 0 && rank == 0) {
    for (int w = 0; w < THREADS / 32; ++w) taken = max(taken, static_cast<int>(s_warp[w]));
    *p.n_free = height - taken;
  }
  if (odd && rank == 0) atomicOr(&g_device_error, ERR_BAD_INDEX);
  // a warp a sequence
  const int w0 = rank * (THREADS / 32) + warp_id(), warps = ctas * (THREADS / 32);
  for (int b = w0; b < p.B; b += warps) {
    const int n = -s_move[b], at = s_at[b];
    int32_t* t = p.table + static_cast<long long>(b) * p.max_pages + s_kept[b];
    for (int e = lane; e < n; e += 32) {
      const int page = t[e];
      page_ok(p, page);
      if (at + e < p.n_pages) p.free_pages[at + e] = page;
      t[e] = -1;
    }
  }
  together();  // the stack is whole
  for (int b = w0; b < p.B; b += warps) {
    const int n = s_move[b], at = s_at[b];
    int32_t* t = p.table + static_cast<long long>(b) * p.max_pages + s_kept[b];
    for (int e = lane; e < n; e += 32) {
      const int page = __ldcg(p.free_pages + at - e);
      if (!page_ok(p, page) && p.granted) p.granted[b] = 0;
      t[e] = page;
    }
  }
  if (!p.slots) return;
  together();  // the table is whole
  for (int row = rank * THREADS + tid; row < p.rows; row += ctas * THREADS) {
    int b, back;
    const bool has = row_seq(p.row_start, p.B, row, b, back);
    p.slots[row] = has ? page_slot(p, b, back, s_kept[b] + max(s_move[b], 0)) : -1;
  }
}

__global__ void __launch_bounds__(256) kv_slots_kernel(const __grid_constant__ PagesParams p) {
  grid_wait();
  const int row = blockIdx.x * 256 + threadIdx.x;
  if (row >= p.rows) return;
  int b, back;
  const bool has = row_seq(p.row_start, p.B, row, b, back);
  p.slots[row] = has ? page_slot(p, b, back, p.held[b]) : -1;
}

static cudaError_t kv_pages(const PagesParams& p, cudaStream_t st, unsigned& kernels) {
  PagesParams first = p;
  const bool apart = p.slots && p.rows > kPagesFew;
  if (apart) first.slots = nullptr;
  const size_t smem = 3 * sizeof(int) * p.B;
  cudaError_t e = cudaSuccess;
  if (pages_one_cta(p)) {
    e = launch_early(kv_pages_kernel<256, 1>, dim3(1), 256, smem, st, first);
  } else {
    e = allow_smem<kv_pages_kernel<1024, 4>>(3 * sizeof(int) * 4096);
    if (e == cudaSuccess) e = launch_early(kv_pages_kernel<1024, 4>, dim3(8), 1024, smem, st, first, 8);
  }
  kernels = apart ? 2 : 1;
  if (apart && e == cudaSuccess) e = launch_early(kv_slots_kernel, dim3((p.rows + 255) / 256), 256, 0, st, p);
  return e;
}

}  // namespace tkb
