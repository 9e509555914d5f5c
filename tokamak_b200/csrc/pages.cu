// pages.cu -- block tables and slot maps from the lengths of the requests.
#include "tkb_common.cuh"
#include "../../include/tkm_b200.h"

namespace tkb {

// Latency bounds it: some 20 bytes a sequence and 8 a page moved.  One launch
// of one cluster: every CTA sums the sequences' needs for itself (two scans over
// at most 4096 of them, in shared memory), so that the CTAs share nothing but
// the order of three phases, kept by cluster barriers: all have read the state;
// surplus pages are on the stack; the missing ones are in the table.
struct PagesParams {
  int32_t* table;
  int32_t* held;
  const int32_t* lens;
  int32_t* free_pages;
  int32_t* n_free;
  int32_t* granted;
  long long* slots;
  const int32_t* row_start;
  int rows, B, max_pages, page_size, n_pages;
};

constexpr int kPagesThreads = 1024;
constexpr int kPagesSeqs = 4;  // sequences per thread of the scans: 4096 in all

// Exclusive sums over the block of each thread's value, and the total.
TKB_DEVFN int pages_scan(int v, int* s_warp, int& total) {
  const int lane = lane_id(), w = warp_id();
  int x = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, d);
    if (lane >= d) x += y;
  }
  __syncthreads();
  if (lane == 31) s_warp[w] = x;
  __syncthreads();
  int sum = s_warp[lane];
  int upto = sum;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, upto, d);
    if (lane >= d) upto += y;
  }
  total = __shfl_sync(0xffffffffu, upto, 31);
  const int before = __shfl_sync(0xffffffffu, upto - sum, w);
  return before + x - v;
}

__global__ void __launch_bounds__(kPagesThreads) kv_pages_kernel(const __grid_constant__ PagesParams p) {
  // per sequence: pages kept, pages to give back (with a minus sign) or to take, and where they go on or come off the stack
  extern __shared__ int s_seq[];
  __shared__ int s_warp[32];
  int* s_kept = s_seq;
  int* s_move = s_seq + p.B;
  int* s_at = s_seq + 2 * p.B;
  const int tid = threadIdx.x, lane = lane_id();
  const int rank = blockIdx.x, ctas = gridDim.x;  // the grid is one cluster
  grid_wait();
  int kept[kPagesSeqs], back[kPagesSeqs], need[kPagesSeqs], sum_back = 0, sum_need = 0;
  bool odd = false, room[kPagesSeqs];
  const long long most = static_cast<long long>(p.max_pages) * p.page_size;
#pragma unroll
  for (int i = 0; i < kPagesSeqs; ++i) {
    const int b = tid * kPagesSeqs + i;
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
  int all_back, all_need;
  int at_back = n_free + pages_scan(sum_back, s_warp, all_back);
  int at_need = pages_scan(sum_need, s_warp, all_need);
  odd |= n_free + all_back > p.n_pages;
  const int height = min(n_free + all_back, p.n_pages);
  cluster_sync();  // all have read held and n_free
  int taken = 0;
#pragma unroll
  for (int i = 0; i < kPagesSeqs; ++i) {
    const int b = tid * kPagesSeqs + i;
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
  if (lane == 0) s_warp[warp_id()] = taken;
  __syncthreads();
  if (tid == 0 && rank == 0) {
    for (int w = 0; w < kPagesThreads / 32; ++w) taken = max(taken, s_warp[w]);
    *p.n_free = height - taken;
  }
  if (odd && rank == 0) atomicOr(&g_device_error, ERR_BAD_INDEX);
  // a warp a sequence
  const int w0 = rank * (kPagesThreads / 32) + warp_id(), warps = ctas * (kPagesThreads / 32);
  for (int b = w0; b < p.B; b += warps) {
    const int n = -s_move[b], at = s_at[b];
    int32_t* t = p.table + static_cast<long long>(b) * p.max_pages + s_kept[b];
    for (int e = lane; e < n; e += 32) {
      if (at + e < p.n_pages) p.free_pages[at + e] = t[e];
      t[e] = -1;
    }
  }
  cluster_sync();  // the stack is whole
  for (int b = w0; b < p.B; b += warps) {
    const int n = s_move[b], at = s_at[b];
    int32_t* t = p.table + static_cast<long long>(b) * p.max_pages + s_kept[b];
    for (int e = lane; e < n; e += 32) t[e] = __ldcg(p.free_pages + at - e);
  }
  if (!p.slots) return;
  cluster_sync();  // the table is whole
  for (int row = rank * kPagesThreads + tid; row < p.rows; row += ctas * kPagesThreads) {
    int b = row, back = 1;
    bool has = true;
    if (p.row_start) {
      int lo = 0, hi = p.B - 1;  // last b with row_start[b] <= row
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (__ldg(p.row_start + mid) <= row) lo = mid;
        else hi = mid - 1;
      }
      b = lo;
      const int end = __ldg(p.row_start + b + 1);
      has = __ldg(p.row_start + b) <= row && row < end;
      back = end - row;
    }
    const long long slot = static_cast<long long>(__ldg(p.lens + b)) - back;
    const int pages = s_kept[b] + max(s_move[b], 0);
    long long to = -1;
    if (has && slot >= 0 && slot < static_cast<long long>(pages) * p.page_size) {
      const int i = static_cast<int>(slot / p.page_size);
      const int page = __ldcg(p.table + static_cast<long long>(b) * p.max_pages + i);
      if (static_cast<unsigned>(page) < static_cast<unsigned>(p.n_pages))
        to = static_cast<long long>(page) * p.page_size + slot % p.page_size;
    }
    p.slots[row] = to;
  }
}

static cudaError_t kv_pages(const PagesParams& p, cudaStream_t st) {
  const int ctas = p.B > 128 || p.rows > 4096 ? 8 : 1;
  const cudaError_t e = allow_smem<kv_pages_kernel>(3 * sizeof(int) * kPagesThreads * kPagesSeqs);
  if (e != cudaSuccess) return e;
  return launch_early(kv_pages_kernel, dim3(ctas), kPagesThreads, 3 * sizeof(int) * p.B, st, p, ctas);
}

}  // namespace tkb
