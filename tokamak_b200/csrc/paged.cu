// paged.cu -- the paged key-value cache: new tokens enter it, one new token
// per sequence attends over it, tokens leave it by accumulated weight.
#include "tkb_common.cuh"
#include "../../include/tkm_b200.h"

namespace tkb {

// Element offset of slot 0 of (page, kv head) in k and v.
TKB_DEVFN long long page_offset(const tkb_kv_cache& c, int page, int h) {
  return static_cast<long long>(page) * c.page_stride + static_cast<long long>(h) * c.page_size * c.D;
}
// Index of (page, kv head, 0) in pos and weight.
TKB_DEVFN long long meta_offset(const tkb_kv_cache& c, int page, int h) {
  return (static_cast<long long>(page) * c.Hkv + h) * c.page_size;
}
// Page `i` of sequence b, or -1 (and the error bit) where the table names none.
TKB_DEVFN int page_of(const tkb_kv_cache& c, int b, int i) {
  const int p = __ldg(c.block_table + static_cast<long long>(b) * c.max_pages + i);
  if (static_cast<unsigned>(p) < static_cast<unsigned>(c.n_pages)) return p;
  atomicOr(&g_device_error, ERR_BAD_INDEX);
  return -1;
}
// Tokens sequence b holds, inside what its table can hold.
TKB_DEVFN int held_of(const tkb_kv_cache& c, int b) {
  const int n = c.seq_lens[b], most = c.max_pages * c.page_size;
  if (n >= 0 && n <= most) return n;
  atomicOr(&g_device_error, ERR_BAD_INDEX);
  return n < 0 ? 0 : most;
}

// ============================================================ lengths
__global__ void kv_lens_kernel(int32_t* __restrict__ lens, int32_t* __restrict__ seen,
                               const int32_t* __restrict__ row_start, int add, int limit, int B) {
  for (int b = blockIdx.x * blockDim.x + threadIdx.x; b < B; b += gridDim.x * blockDim.x) {
    const int n = row_start ? row_start[b + 1] - row_start[b] : add;
    const long long next = static_cast<long long>(lens[b]) + n;
    if (n > 0 && next > limit) atomicOr(&g_device_error, ERR_BAD_INDEX);
    lens[b] = static_cast<int>(next < limit ? next : limit);
    if (seen) seen[b] += n;
  }
}

// ============================================================ append
// qkv_prep_fwd_kernel (rows.cu) with each row's own position, its K and V
// columns stored to the row's slot.  One block per row; the row's D/2 cosines
// and sines are computed once, in shared memory, for all its heads.
struct AppendParams {
  tkb_kv_cache c;
  const void* qkv;
  long long qkv_stride;
  const float* bias;
  const float* gain;
  void* out;
  long long out_stride;
  const int32_t* row_start;
  const int32_t* seen;
  int out_full, rows, Hq, qknorm, rope;
  RopeTable tab;
};

template <typename T>
__global__ void __launch_bounds__(NT) kv_append_kernel(const __grid_constant__ AppendParams p) {
  __shared__ float s_cs[64], s_sn[64];
  __shared__ long long s_kv, s_meta;  // element offset of the row's slot of kv head 0; its pos / weight index
  __shared__ int s_pos;
  const tkb_kv_cache& c = p.c;
  const int Hq = p.Hq, Hkv = c.Hkv, D = c.D, C = (Hq + 2 * Hkv) * D, nqk = Hq + Hkv, nvec = C / 8, grp = D / 8;
  const T* in = static_cast<const T*>(p.qkv);
  T* out = static_cast<T*>(p.out);
  for (int row = blockIdx.x; row < p.rows; row += gridDim.x) {
    __syncthreads();  // the previous row's shared values have been read
    if (threadIdx.x < D / 2) {
      // the row's sequence: the last b with row_start[b] <= row
      int b = row, back = 1;
      bool has = true;
      if (p.row_start) {
        int lo = 0, hi = c.B;
        while (hi - lo > 1) {
          const int mid = (lo + hi) >> 1;
          if (p.row_start[mid] <= row) lo = mid; else hi = mid;
        }
        b = lo;
        back = p.row_start[b + 1] - row;
        has = back > 0 && p.row_start[b] <= row;
      }
      const int slot = c.seq_lens[b] - back;
      const int pos = (p.seen ? p.seen[b] : c.seq_lens[b]) - back;
      if (p.rope) {
        float sn, cs;
        rope_cs(pos, p.tab.inv_freq[threadIdx.x], sn, cs);
        s_cs[threadIdx.x] = cs;
        s_sn[threadIdx.x] = sn;
      }
      if (threadIdx.x == 0) {
        int page = -1;
        if (has && slot >= 0 && slot < c.max_pages * c.page_size) page = page_of(c, b, slot / c.page_size);
        else atomicOr(&g_device_error, ERR_BAD_INDEX);
        const int in_page = slot % c.page_size;
        s_kv = page < 0 ? -1 : page_offset(c, page, 0) + static_cast<long long>(in_page) * D;
        s_meta = page < 0 ? -1 : meta_offset(c, page, 0) + in_page;
        s_pos = pos;
      }
    }
    __syncthreads();
    const long long base = static_cast<long long>(row) * p.qkv_stride;
    for (int v0 = 0; v0 < nvec; v0 += NT) {
      const int vi = v0 + threadIdx.x;
      const bool act = vi < nvec;
      const int col = vi * 8, hd = col / D, d = col % D;
      float v[8];
      if (act) {
        ldv<T, 8>(in + base + col, v);
        if (p.bias) {
          float bb[8];
          ldf<8>(p.bias + col, bb);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] += bb[e];
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = 0.f;
      }
      if (p.qknorm) {
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(v[e], v[e], ss);
        for (int m = grp >> 1; m >= 1; m >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, m);
        if (act && hd < nqk) {
          const float is = 1.0f / sqrtf(ss / static_cast<float>(D) + 1e-5f);
          float gg[8];
          if (p.gain) ldf<8>(p.gain + col, gg);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = v[e] * is * (p.gain ? gg[e] : 1.0f);
        }
      }
      if (!act) continue;
      if (p.rope && hd < nqk) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float sn = s_sn[d / 2 + e], cs = s_cs[d / 2 + e];
          const float x0 = v[2 * e], x1 = v[2 * e + 1];
          v[2 * e] = x0 * cs - x1 * sn;
          v[2 * e + 1] = x0 * sn + x1 * cs;
        }
      }
      if (out && (hd < Hq || p.out_full)) stv<T, 8>(out + static_cast<long long>(row) * p.out_stride + col, v);
      if (hd >= Hq && s_kv >= 0) {
        const int h = hd < nqk ? hd - Hq : hd - nqk;
        T* pool = static_cast<T*>(hd < nqk ? c.k : c.v);
        stv<T, 8>(pool + s_kv + static_cast<long long>(h) * c.page_size * D + d, v);
      }
    }
    if (s_meta >= 0)
      for (int h = threadIdx.x; h < Hkv; h += NT) {
        const long long at = s_meta + static_cast<long long>(h) * c.page_size;
        if (c.pos) c.pos[at] = s_pos;
        if (c.weight) c.weight[at] = 0.f;
      }
  }
}

template <typename T>
static cudaError_t kv_append_t(const AppendParams& p, cudaStream_t st) {
  kv_append_kernel<T><<<row_grid(p.rows, 8), NT, 0, st>>>(p);
  return cudaGetLastError();
}

// ============================================================ attention of one token
struct DecodeParams {
  tkb_kv_cache c;
  const void* q;
  long long q_stride;
  void* out;
  long long out_stride;
  float* lse;
  int Hq, accumulate;
  float scale_log2;
};

// One block per (sequence, kv head); a warp per key, lanes over D.
template <typename T, int D>
__global__ void __launch_bounds__(128) paged_decode_kernel(const __grid_constant__ DecodeParams p) {
  constexpr int W = 4, E = D / 32;
  __shared__ float s_m[W], s_l[W], s_o[W][D];
  const tkb_kv_cache& c = p.c;
  const int b = blockIdx.x / c.Hkv, h = blockIdx.x % c.Hkv, G = p.Hq / c.Hkv;
  const int n = held_of(c, b), w = warp_id(), lane = lane_id();
  const T* K = static_cast<const T*>(c.k);
  const T* V = static_cast<const T*>(c.v);
  for (int g = 0; g < G; ++g) {
    const int hq = h * G + g;
    float q[E], o[E], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      q[e] = Elem<T>::ld(static_cast<const T*>(p.q) + b * p.q_stride + hq * D + lane * E + e) * p.scale_log2;
      o[e] = 0.f;
    }
    for (int j = w; j < n; j += W) {
      const int page = page_of(c, b, j / c.page_size);
      if (page < 0) continue;
      const long long at = page_offset(c, page, h) + static_cast<long long>(j % c.page_size) * D + lane * E;
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) s = fmaf(q[e], Elem<T>::ld(K + at + e), s);
      s = warp_sum(s);
      const float mn = fmaxf(m, s), keep = m == -INFINITY ? 0.f : exp2f(m - mn), pr = exp2f(s - mn);
      l = l * keep + pr;
      m = mn;
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = fmaf(pr, Elem<T>::ld(V + at + e), o[e] * keep);
    }
    __syncthreads();
    if (lane == 0) {
      s_m[w] = m;
      s_l[w] = l;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) s_o[w][lane * E + e] = o[e];
    __syncthreads();
    float M = -INFINITY, Lsum = 0.f;
    for (int i = 0; i < W; ++i) M = fmaxf(M, s_m[i]);
    for (int i = 0; i < W; ++i) Lsum += s_m[i] == -INFINITY ? 0.f : s_l[i] * exp2f(s_m[i] - M);
    const float lse2 = M == -INFINITY ? -INFINITY : M + log2f(Lsum);
    for (int d = threadIdx.x; d < D; d += 128) {
      float acc = 0.f;
      for (int i = 0; i < W; ++i) acc += s_m[i] == -INFINITY ? 0.f : s_o[i][d] * exp2f(s_m[i] - M);
      Elem<T>::st(static_cast<T*>(p.out) + b * p.out_stride + hq * D + d, M == -INFINITY ? 0.f : acc / Lsum);
    }
    if (threadIdx.x == 0 && p.lse) p.lse[b * p.Hq + hq] = lse2 * 0.6931471805599453f;
    if (p.accumulate)
      for (int j = w; j < n; j += W) {
        const int page = page_of(c, b, j / c.page_size);
        if (page < 0) continue;
        const int in_page = j % c.page_size;
        const long long at = page_offset(c, page, h) + static_cast<long long>(in_page) * D + lane * E;
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) s = fmaf(q[e], Elem<T>::ld(K + at + e), s);
        s = warp_sum(s);
        if (lane == 0) c.weight[meta_offset(c, page, h) + in_page] += exp2f(s - lse2);
      }
  }
}

template <typename T>
static cudaError_t paged_decode_t(const DecodeParams& p, cudaStream_t st) {
  const int grid = p.c.B * p.c.Hkv;
  if (p.c.D == 64) paged_decode_kernel<T, 64><<<grid, 128, 0, st>>>(p);
  else paged_decode_kernel<T, 128><<<grid, 128, 0, st>>>(p);
  return cudaGetLastError();
}

// ============================================================ eviction
struct EvictParams {
  tkb_kv_cache c;
  const int32_t* seen;
  int32_t* lists;  // per (sequence, kv head): `cap` destinations, then `cap` sources
  int budget, recent, sinks, cap;
};

// Floats as unsigned numbers of the same order (-0 as +0, NaN below -inf).
TKB_DEVFN uint32_t order_key(float x) {
  if (x != x) return 0u;
  const uint32_t u = __float_as_uint(x + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Inclusive block-wide prefix sum (blockDim.x = 1024); `sh` holds 32 ints.
TKB_DEVFN int block_scan(int v, int* sh, int& total) {
  const int lane = lane_id(), w = warp_id();
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, v, d);
    if (lane >= d) v += t;
  }
  __syncthreads();
  if (lane == 31) sh[w] = v;
  __syncthreads();
  int pre = 0, all = 0;
  for (int i = 0; i < 32; ++i) {
    const int t = sh[i];
    if (i < w) pre += t;
    all += t;
  }
  total = all;
  return v + pre;
}

template <typename T>
__global__ void __launch_bounds__(1024) kv_evict_kernel(const __grid_constant__ EvictParams p) {
  __shared__ int hist[256], sh[32], s_bin, s_need;
  const tkb_kv_cache& c = p.c;
  const int b = blockIdx.x / c.Hkv, h = blockIdx.x % c.Hkv, tid = threadIdx.x;
  const int n = held_of(c, b);
  if (n <= p.budget) return;
  const int newest = p.seen[b] - p.recent;
  auto key_of = [&](int j) -> uint32_t {
    const int page = page_of(c, b, j / c.page_size);
    if (page < 0) return 0u;
    const long long at = meta_offset(c, page, h) + j % c.page_size;
    const int pos = c.pos[at];
    if (pos >= newest || pos < p.sinks) return 0xFFFFFFFFu;
    return order_key(c.weight[at]);
  };
  // the budget-th largest key, eight bits at a time
  uint32_t prefix = 0, mask = 0;
  int need = p.budget;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += 1024) hist[i] = 0;
    __syncthreads();
    for (int j = tid; j < n; j += 1024) {
      const uint32_t k = key_of(j);
      if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & 255], 1);
    }
    __syncthreads();
    if (tid == 0) {
      int above = 0, bin = 255;
      while (above + hist[bin] < need) above += hist[bin--];
      s_bin = bin;
      s_need = need - above;
    }
    __syncthreads();
    prefix |= static_cast<uint32_t>(s_bin) << shift;
    mask |= 255u << shift;
    need = s_need;
    __syncthreads();
  }
  // freed slots below the budget, kept tokens at it and above, both ascending
  int32_t* to = p.lists + static_cast<long long>(blockIdx.x) * 2 * p.cap;
  int32_t* from = to + p.cap;
  int ties = 0, holes = 0, movers = 0;
  for (int j0 = 0; j0 < n; j0 += 1024) {
    const int j = j0 + tid;
    const uint32_t k = j < n ? key_of(j) : 0u;
    const bool tie = j < n && k == prefix;
    int total;
    const int rank = ties + block_scan(tie, sh, total) - tie;
    ties += total;
    const bool kept = j < n && (k > prefix || (tie && rank < need));
    const bool hole = j < n && j < p.budget && !kept, mover = kept && j >= p.budget;
    const int at = holes + block_scan(hole, sh, total) - hole;
    holes += total;
    if (hole) to[at] = j;
    const int am = movers + block_scan(mover, sh, total) - mover;
    movers += total;
    if (mover) from[am] = j;
  }
  __syncthreads();
  const int vecs = c.D * static_cast<int>(sizeof(T)) / 16;
  for (int i = warp_id(); i < movers; i += 32) {
    const int dj = to[i], sj = from[i];
    const int dp = page_of(c, b, dj / c.page_size), sp = page_of(c, b, sj / c.page_size);
    if (dp < 0 || sp < 0) continue;
    const long long d0 = page_offset(c, dp, h) + static_cast<long long>(dj % c.page_size) * c.D;
    const long long s0 = page_offset(c, sp, h) + static_cast<long long>(sj % c.page_size) * c.D;
    for (int v = lane_id(); v < 2 * vecs; v += 32) {
      T* pool = static_cast<T*>(v < vecs ? c.k : c.v);
      const int o = v < vecs ? v : v - vecs;
      reinterpret_cast<uint4*>(pool + d0)[o] = reinterpret_cast<const uint4*>(pool + s0)[o];
    }
    if (lane_id() == 0) {
      const long long dm = meta_offset(c, dp, h) + dj % c.page_size, sm = meta_offset(c, sp, h) + sj % c.page_size;
      c.pos[dm] = c.pos[sm];
      c.weight[dm] = c.weight[sm];
    }
  }
}

template <typename T>
static cudaError_t kv_evict_t(const EvictParams& p, cudaStream_t st) {
  kv_evict_kernel<T><<<p.c.B * p.c.Hkv, 1024, 0, st>>>(p);
  return cudaGetLastError();
}

}  // namespace tkb
