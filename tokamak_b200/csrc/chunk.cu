// chunk.cu -- attention of a chunk of new tokens over the paged key-value
// cache: pieces of prompts, whole prompts, drafted tokens, single tokens.
#include "tkb_common.cuh"
#include "../../include/tkm_b200.h"

namespace tkb {

struct ChunkParams {
  tkb_kv_cache c;
  const void* q;
  void* out;
  float* lse;
  const int32_t* row_start;
  long long q_stride, out_stride;
  int rows, Hq, G;
  float scale_log2;
};

// The rows of sequence b: first row and number, inside [0, rows).
TKB_DEVFN void chunk_rows(const int32_t* row_start, int rows, int b, int& first, int& n) {
  if (!row_start) {
    first = b;
    n = 1;
    return;
  }
  int lo = row_start[b], hi = row_start[b + 1];
  if (lo < 0 || hi < lo || hi > rows) {
    atomicOr(&g_device_error, ERR_BAD_INDEX);
    lo = min(max(lo, 0), rows);
    hi = min(max(hi, lo), rows);
  }
  first = lo;
  n = hi - lo;
}

template <typename T, int E>
TKB_DEVFN void lane_values(const T* p, float (&f)[E]) {
#pragma unroll
  for (int e = 0; e < E; ++e) f[e] = static_cast<float>(p[e]);
}

// One query row of one head by a warp, slot by slot.
template <typename T, int D>
__global__ void __launch_bounds__(256) chunk_simple_kernel(const __grid_constant__ ChunkParams p) {
  constexpr int E = D / 32;
  const int lane = lane_id(), row = blockIdx.x;
  const tkb_kv_cache& c = p.c;
  grid_wait();
  int b = row, first = row, n = 1;
  if (p.row_start) {
    int lo = 0, hi = c.B;  // last b with row_start[b] <= row
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (p.row_start[mid] <= row) lo = mid;
      else hi = mid - 1;
    }
    b = lo;
    if (b >= c.B) return;
    chunk_rows(p.row_start, p.rows, b, first, n);
    if (row < first || row >= first + n) return;
  }
  const int held = c.seq_lens[b], most = c.max_pages * c.page_size;
  int upto = held - n + (row - first) + 1;  // slots this row sees
  if (upto <= 0 || upto > most) {
    if (lane == 0) atomicOr(&g_device_error, ERR_BAD_INDEX);
    upto = min(max(upto, 0), most);
  }
  for (int hq = warp_id(); hq < p.Hq; hq += 8) {
    const int h = hq / p.G;
    float q[E], o[E], m = -INFINITY, l = 0.f;
    lane_values(static_cast<const T*>(p.q) + row * p.q_stride + static_cast<long long>(hq) * D + lane * E, q);
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = 0.f;
    int page = -1;
    for (int j = 0; j < upto; ++j) {
      const int in = j % c.page_size;
      if (in == 0) page = page_of(c, b, j / c.page_size);
      if (page < 0) continue;
      const long long at = page_offset(c, page, h) + static_cast<long long>(in) * D + lane * E;
      float k[E], v[E], s = 0.f;
      lane_values(static_cast<const T*>(c.k) + at, k);
      lane_values(static_cast<const T*>(c.v) + at, v);
#pragma unroll
      for (int e = 0; e < E; ++e) s = fmaf(q[e], k[e], s);
      s = warp_sum(s) * p.scale_log2;
      const float mn = fmaxf(m, s), base = mn == -INFINITY ? 0.f : mn;
      const float f = ex2(m - base), w = ex2(s - base);
      l = l * f + w;
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = fmaf(w, v[e], o[e] * f);
      m = mn;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    T* out = static_cast<T*>(p.out) + row * p.out_stride + static_cast<long long>(hq) * D + lane * E;
#pragma unroll
    for (int e = 0; e < E; ++e) out[e] = static_cast<T>(o[e] * inv);
    if (p.lse && lane == 0) p.lse[static_cast<long long>(row) * p.Hq + hq] = (m + lg2(l)) * 0.6931471805599453f;
  }
}

template <typename T>
static cudaError_t paged_chunk_t(const ChunkParams& p, cudaStream_t st) {
  if (p.c.D == 64) return launch_early(chunk_simple_kernel<T, 64>, dim3(p.rows), 256, 0, st, p);
  return launch_early(chunk_simple_kernel<T, 128>, dim3(p.rows), 256, 0, st, p);
}

}  // namespace tkb
