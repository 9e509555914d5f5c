// paged.cu -- the paged key-value cache: new tokens enter it, one new token
// per sequence attends over it, tokens leave it by accumulated weight.
#include <atomic>

#include "tkb_common.cuh"
#include "../../include/tkm_b200.h"

namespace tkb {

// Raises a kernel's limit of dynamic shared memory, once per device (the call
// costs as much host time as a launch).
template <auto Kernel>
static cudaError_t allow_smem(int bytes) {
  static std::atomic<unsigned long long> done{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const unsigned long long bit = dev < 64 ? 1ull << dev : 0;
  if (done.load(std::memory_order_relaxed) & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

// Launches of this file and sample.cu let the kernel come up while the one
// before it in the stream ends (programmatic dependent launch): the kernel's
// first act is grid_wait(), which returns when everything launched before has
// completed and is visible, so nothing else changes.
TKB_DEVFN void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <typename P>
static cudaError_t launch_early(void (*kernel)(P), dim3 grid, int block, size_t smem, cudaStream_t st, const P& p,
                                int cluster = 0) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

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
// columns stored to the row's slot.  HBM bounds it for prompts.  A block takes
// R * GROUPS rows: where they go and their cosines and sines (D/2 each, for
// all heads) are found once, in shared memory, while the first columns load;
// then a thread walks R rows of a column at a time, so that bias and gain are
// read once for them, with the next R loads in flight.  At 12.5 k rows of 10240
// f16 columns (563 MB): 2 x 2 rows 115 us (0.75 of HBM), 2 x 1 119, 4 x 1 124,
// 1 x 4 125, 2 x 4 127, 4 x 2 149 (fewer, larger blocks leave a ragged last
// wave).  One row a block when the rows would not fill the GPU.
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

// Eight elements as loaded, and as floats.
template <typename T>
struct Raw8 {
  uint4 q[sizeof(T) / 2];
  TKB_DEVFN void load(const T* p) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) q[i] = ld_stream_v4(reinterpret_cast<const uint4*>(p) + i);
  }
  TKB_DEVFN void floats(float (&f)[8]) const {
    const uint32_t u[4] = {q[0].x, q[0].y, q[0].z, q[0].w};
    if constexpr (sizeof(T) == 4) {
      const uint32_t v[4] = {q[1].x, q[1].y, q[1].z, q[1].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        f[i] = __uint_as_float(u[i]);
        f[4 + i] = __uint_as_float(v[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 x = unpack2<std::is_same<T, __nv_bfloat16>::value>(u[i]);
        f[2 * i] = x.x;
        f[2 * i + 1] = x.y;
      }
    }
  }
};

template <typename T, int D, int R, int GROUPS>
__global__ void __launch_bounds__(NT) kv_append_kernel(const __grid_constant__ AppendParams p) {
  constexpr int RB = R * GROUPS;  // rows of the block
  __shared__ float s_cs[RB][64], s_sn[RB][64];
  __shared__ long long s_kv[RB], s_meta[RB];  // element offset of the row's slot of kv head 0; its pos / weight index
  __shared__ int s_pos[RB];
  const tkb_kv_cache& c = p.c;
  const int Hq = p.Hq, Hkv = c.Hkv, C = (Hq + 2 * Hkv) * D, nqk = Hq + Hkv, nvec = C / 8;
  constexpr int grp = D / 8;
  const T* in = static_cast<const T*>(p.qkv);
  T* out = static_cast<T*>(p.out);
  const int row0 = blockIdx.x * RB, tid = threadIdx.x, rows = min(RB, p.rows - row0);
  in += static_cast<long long>(row0) * p.qkv_stride;
  if (out) out += static_cast<long long>(row0) * p.out_stride;
  // the next column's loads are under way while one is worked on, the first one's during what comes before
  grid_wait();
  Raw8<T> raw[R];
  auto fetch = [&](int g, int vi) {
    if (vi < nvec)
#pragma unroll
      for (int r = 0; r < R; ++r)
        if (g + r < rows) raw[r].load(in + (g + r) * p.qkv_stride + vi * 8);
  };
  fetch(0, tid);
  // ---- where the rows go: the sequence is the last b with row_start[b] <= row
  int b0 = row0;
  if (p.row_start) {
    int upto = 0;
    for (int b = 0; b < c.B; b += NT) upto += __syncthreads_count(b + tid < c.B && p.row_start[b + tid] <= row0);
    b0 = upto - 1;
  }
  if (tid < rows) {
    const int row = row0 + tid;
    int b = p.row_start ? b0 : row, back = 1;
    bool has = true;
    if (p.row_start) {
      while (b + 1 < c.B && p.row_start[b + 1] <= row) ++b;
      has = b >= 0 && p.row_start[b] <= row && row < p.row_start[b + 1];
      b = max(b, 0);
      back = p.row_start[b + 1] - row;
    }
    const int held = c.seq_lens[b], slot = held - back;
    int page = -1;
    if (!has || !p.seen || p.seen[b] >= 0) {  // else the sequence takes no part
      if (has && slot >= 0 && slot < c.max_pages * c.page_size) page = page_of(c, b, slot / c.page_size);
      else atomicOr(&g_device_error, ERR_BAD_INDEX);
    }
    const int in_page = slot % c.page_size;
    s_kv[tid] = page < 0 ? -1 : page_offset(c, page, 0) + static_cast<long long>(in_page) * D;
    s_meta[tid] = page < 0 ? -1 : meta_offset(c, page, 0) + in_page;
    s_pos[tid] = (p.seen ? p.seen[b] : held) - back;
  }
  __syncthreads();
  if (p.rope) {
    for (int i = tid; i < RB * (D / 2); i += NT) {
      const int r = i / (D / 2), d = i % (D / 2);
      float sn = 0.f, cs = 1.f;
      if (r < rows) rope_cs(s_pos[r], p.tab.inv_freq[d], sn, cs);
      s_cs[r][d] = cs;
      s_sn[r][d] = sn;
    }
    __syncthreads();
  }
#pragma unroll 1
  for (int g = 0; g < rows; g += R)
#pragma unroll 1
  for (int v0 = 0; v0 < nvec; v0 += NT) {
    const int vi = v0 + tid;
    const bool act = vi < nvec;
    const int col = vi * 8, hd = col / D, d = col % D;
    float v[R][8], bb[8], gg[8];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (act && g + r < rows) raw[r].floats(v[r]);
      else
#pragma unroll
        for (int e = 0; e < 8; ++e) v[r][e] = 0.f;
    }
    if (v0 + NT < nvec) fetch(g, vi + NT);
    else if (g + R < rows) fetch(g + R, tid);
    if (p.bias && act) {
      ldf<8>(p.bias + col, bb);
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int e = 0; e < 8; ++e) v[r][e] += bb[e];
    }
    const bool turned = act && hd < nqk;
    if (p.qknorm) {
#pragma unroll
      for (int e = 0; e < 8; ++e) gg[e] = 1.0f;
      if (p.gain && turned) ldf<8>(p.gain + col, gg);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(v[r][e], v[r][e], ss);
#pragma unroll
        for (int m = grp >> 1; m >= 1; m >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, m);
        if (turned) {
          const float is = rsqrtf(fmaf(ss, 1.0f / D, 1e-5f));
#pragma unroll
          for (int e = 0; e < 8; ++e) v[r][e] *= is * gg[e];
        }
      }
    }
    if (!act) continue;
    // the column's place in a slot's K or V, for the columns that have one
    T* pool = static_cast<T*>(turned ? c.k : c.v) + static_cast<long long>(turned ? hd - Hq : hd - nqk) * c.page_size * D + d;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (g + r >= rows) break;
      if (p.rope && turned) {
        const float4 cs = *reinterpret_cast<const float4*>(&s_cs[g + r][d / 2]),
                     sn = *reinterpret_cast<const float4*>(&s_sn[g + r][d / 2]);
        const float c4[4] = {cs.x, cs.y, cs.z, cs.w}, s4[4] = {sn.x, sn.y, sn.z, sn.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x0 = v[r][2 * e], x1 = v[r][2 * e + 1];
          v[r][2 * e] = x0 * c4[e] - x1 * s4[e];
          v[r][2 * e + 1] = x0 * s4[e] + x1 * c4[e];
        }
      }
      if (out && (hd < Hq || p.out_full)) stv<T, 8>(out + (g + r) * p.out_stride + col, v[r]);
      if (hd >= Hq && s_kv[g + r] >= 0) stv<T, 8>(pool + s_kv[g + r], v[r]);
    }
  }
  for (int i = tid; i < RB * Hkv; i += NT) {
    const int r = i % RB, h = i / RB;
    if (r >= rows || s_meta[r] < 0) continue;
    const long long at = s_meta[r] + static_cast<long long>(h) * c.page_size;
    if (c.pos) c.pos[at] = s_pos[r];
    if (c.weight) c.weight[at] = 0.f;
  }
}

template <typename T, int D>
static cudaError_t kv_append_d(const AppendParams& p, cudaStream_t st) {
  if (p.rows >= 148 * 8) return launch_early(kv_append_kernel<T, D, 2, 2>, dim3((p.rows + 3) / 4), NT, 0, st, p);
  return launch_early(kv_append_kernel<T, D, 1, 1>, dim3(p.rows), NT, 0, st, p);
}

template <typename T>
static cudaError_t kv_append_t(const AppendParams& p, cudaStream_t st) {
  return p.c.D == 64 ? kv_append_d<T, 64>(p, st) : kv_append_d<T, 128>(p, st);
}

// ============================================================ attention of one token
// out = softmax(scale q K^T) V for one query row per sequence: every cached K
// and V value is read once and used by the G query heads of its kv head, so
// HBM bounds it (4 G FLOP per element read) and the kernel is built around
// keeping loads in flight.
//
// The keys of a unit (sequence, kv head, block of up to 16 query heads) are cut
// into tiles of 16 (8 for fp32 rows of 512 bytes).  All units' tiles, in order,
// are dealt out as equal runs, whatever the lengths: to the CTAs, one per SM,
// and inside a CTA to its warps, each with its own ring of cp.async buffers and
// its own running maximum and sum.  A unit that lies inside one warp's run is
// written by that warp at once; the others are parts, at most two per warp,
// which meet once, at the CTA's end, and where a unit spans CTAs, in the CTA
// that finishes last (a counter in the workspace), in the order of the run, so
// the result does not depend on who that is.  The counter is that of the CTA
// the unit starts in, of which it is the last unit: one per CTA, in one place
// whatever the cache's shape, so that a workspace serves them all in turn.
//
// Measured: 16 sequences of 15-16 k tokens, 64/8 heads of 128, bf16 (1.05 GB):
// 183 us, 5.7 TB/s, 0.88 of HBM, and 17 us for the weights of `accumulate`; 32
// sequences up to 2048, 32/8 heads of 64 (69 MB): 25 us, 10 of them in the tile
// loop; 3 fp32 sequences up to 4097, 16 heads of 128 (127 MB): 29 us.  A block
// per (sequence, kv head) took 67.6 ms, 1491 us and 1723 us.
constexpr int QT = 16;                // query heads per unit (rows of the m16n8k16 product)

struct DecodeParams {
  tkb_kv_cache c;
  const void* q;
  long long q_stride;
  void* out;
  long long out_stride;
  float* lse;
  int Hq, G, qblocks, accumulate;
  float scale_log2;
  int* counters;                      // per CTA, for the unit that goes on from it; 0 between calls
  float* part;                        // [2 * grid][QT][D + 2]: O, then m, l of each row
  float* head;                        // [grid * 16 warps][QT][D]: first parts, when they are not in shared memory
  float* lse2;                        // accumulate: [B][Hq], in powers of 2
  float* scores;                      // accumulate: [B][Hq][cap], in powers of 2
};

template <int D, int ES, int GT>
struct DecodeTile {
  static constexpr int RB = D * ES;                 // bytes of a row
  static constexpr int TK = RB <= 256 ? 16 : 8;     // keys per tile
  static constexpr int HALF = TK * RB;              // bytes of the K (or V) part
  static constexpr int WARPS = D * ES == 128 ? 16 : 8;
  static constexpr int STAGES = ES == 4 && GT > 4 ? 2 : 3;
  static constexpr int RING = STAGES * 2 * HALF;    // per warp
  static constexpr int HEAD = GT <= 8 ? GT * D * 4 : 0;                  // per warp: its first part (else in the workspace)
  static constexpr int EXTRA = ES == 4 ? GT * D * 4 + GT * TK * 4 : 0;   // per warp: q, p
  static constexpr int SMEM = WARPS * (RING + HEAD + EXTRA);
};

// Where a flattened tile index lies.
struct TileAt {
  int b, u, j;   // sequence, (kv head, query block), tile of the unit
  int n, nt;     // tokens held, tiles (at least one, so that an empty sequence gets its zeros)
};
template <int TK>
TKB_DEVFN void tile_seq(const tkb_kv_cache& c, TileAt& t) {
  t.n = t.b < c.B ? held_of(c, t.b) : 0;
  t.nt = max(1, (t.n + TK - 1) / TK);
}
TKB_DEVFN void cp_async16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
TKB_DEVFN void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
TKB_DEVFN void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
TKB_DEVFN void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
TKB_DEVFN void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
template <bool BF16>
TKB_DEVFN void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (BF16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

TKB_DEVFN void decode_lse(const DecodeParams& p, int b, int hq, float M, float L) {
  const float lse2 = M + lg2(L);  // -inf + -inf when nothing is held
  if (p.lse) p.lse[static_cast<long long>(b) * p.Hq + hq] = lse2 * 0.6931471805599453f;
  if (p.accumulate) p.lse2[static_cast<long long>(b) * p.Hq + hq] = lse2;
}
// O is kept times this: f16 probabilities go into the product as multiples of
// 2^-24, which beside a largest of 2^15 are small enough to be added to each.
template <typename T>
constexpr float kPUp = std::is_same<T, __half>::value ? 32768.f : 1.f;
// One finished output row: lane holds columns lane*E ..
template <typename T, int E>
TKB_DEVFN void decode_store(const DecodeParams& p, int b, int hq, int lane, float M, float L, const float (&acc)[E]) {
  constexpr int D = 32 * E;
  const float inv = L == 0.f ? 0.f : 1.0f / (L * kPUp<T>);  // nothing held: zeros
  T* out = static_cast<T*>(p.out) + b * p.out_stride + static_cast<long long>(hq) * D + lane * E;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int e = 0; e < E; ++e) out[e] = acc[e] * inv;
  } else {
    constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
#pragma unroll
    for (int e = 0; e < E; e += 2)
      *reinterpret_cast<uint32_t*>(out + e) = pack2<BF16>(acc[e] * inv, acc[e + 1] * inv);
  }
  if (lane == 0) decode_lse(p, b, hq, M, L);
}

// Byte offset of 16-byte chunk `ch` of row `r` inside a tile half: the chunk
// index is xored with the row so that eight rows' equal chunks (ldmatrix) lie
// in eight different bank groups.
template <int RB>
TKB_DEVFN int swz(int r, int ch) {
  return r * RB + ((ch ^ (r & 7)) << 4);
}

// The 16-bit tile: S = Q K^T and O += P V on m16n8k16 with the query heads as
// the 16 rows (rows past G are zero).  Thread t holds rows t/4 and t/4 + 8.
template <typename T, int D, int GT>
struct TileMma {
  static constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
  using Cfg = DecodeTile<D, 2, GT>;
  static constexpr int GROUP = GT;
  uint32_t q[D / 16][4];
  float o[D / 8][4];
  float m[2], l[2];

  // Two probabilities as 16-bit pairs, times kPUp: rounded towards zero, and the rest; `least` (the smallest normal
  // number, of f16 the smallest of all) at least
  static TKB_DEVFN void split(float p0, float p1, uint32_t& a, uint32_t& b) {
    const float least = BF16 ? 1.17549435e-38f : 5.9604645e-8f;
    p0 = fmaxf(p0 * kPUp<T>, least);
    p1 = fmaxf(p1 * kPUp<T>, least);
    if constexpr (BF16) a = __byte_perm(__float_as_uint(p0), __float_as_uint(p1), 0x7632);
    else asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(a) : "f"(p1), "f"(p0));
    const float2 h = unpack2<BF16>(a);
    b = pack2<BF16>(fmaxf(p0 - h.x, least), fmaxf(p1 - h.y, least));
  }

  TKB_DEVFN void start(const DecodeParams& p, int b, int h0, int rows, uint8_t*) {
    const int r = lane_id() >> 2, c = lane_id() & 3;
    const T* src = static_cast<const T*>(p.q) + b * p.q_stride + static_cast<long long>(h0 + r) * D + 2 * c;
#pragma unroll
    for (int k = 0; k < D / 16; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        q[k][i] = r + (i & 1) * 8 < rows
                      ? __ldg(reinterpret_cast<const uint32_t*>(src + (i & 1) * 8 * D + k * 16 + (i >> 1) * 8))
                      : 0u;
#pragma unroll
    for (int d = 0; d < D / 8; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[d][i] = 0.f;
    m[0] = m[1] = -INFINITY;
    l[0] = l[1] = 0.f;
  }

  // `scores`: where the tile's scores of query head h0 go, or null
  TKB_DEVFN void tile(const DecodeParams& p, const uint8_t* buf, uint8_t*, int valid, int rows, float* scores,
                      long long score_stride) {
    const int lane = lane_id(), mi = lane >> 3, ri = lane & 7;
    const uint32_t kb = smem_u32(buf), vb = kb + Cfg::HALF;
    float s[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int k = 0; k < D / 16; ++k) {
      uint32_t f[4];
      ldsm4(kb + swz<Cfg::RB>((mi >> 1) * 8 + ri, k * 2 + (mi & 1)), f);
      mma16816<BF16>(s[0], q[k], f[0], f[1]);
      mma16816<BF16>(s[1], q[k], f[2], f[3]);
    }
    const int c = 2 * (lane & 3);
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[t][i] *= p.scale_log2;
        if (valid < 16 && t * 8 + c + (i & 1) >= valid) s[t][i] = -INFINITY;
      }
    if (scores) {
      const int r = lane >> 2;
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (r + 8 * i < rows) {
          float* at = scores + (r + 8 * i) * score_stride + c;
          *reinterpret_cast<float2*>(at) = make_float2(s[0][2 * i], s[0][2 * i + 1]);
          *reinterpret_cast<float2*>(at + 8) = make_float2(s[1][2 * i], s[1][2 * i + 1]);
        }
    }
    float mn[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float x = fmaxf(fmaxf(s[0][2 * i], s[0][2 * i + 1]), fmaxf(s[1][2 * i], s[1][2 * i + 1]));
      x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
      x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
      mn[i] = fmaxf(m[i], x);
    }
    if (__any_sync(0xffffffffu, mn[0] > m[0] || mn[1] > m[1])) {
      // a maximum of -inf stays -inf only while nothing was seen: l and o are 0 then
      const float k0 = m[0] == -INFINITY ? 0.f : ex2(m[0] - mn[0]), k1 = m[1] == -INFINITY ? 0.f : ex2(m[1] - mn[1]);
      l[0] *= k0;
      l[1] *= k1;
#pragma unroll
      for (int d = 0; d < D / 8; ++d) {
        o[d][0] *= k0;
        o[d][1] *= k0;
        o[d][2] *= k1;
        o[d][3] *= k1;
      }
      m[0] = mn[0];
      m[1] = mn[1];
    }
    const float m0 = m[0] == -INFINITY ? 0.f : m[0], m1 = m[1] == -INFINITY ? 0.f : m[1];
    uint32_t a[4], b[4];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const float p0 = ex2(s[t][0] - m0), p1 = ex2(s[t][1] - m0), p2 = ex2(s[t][2] - m1), p3 = ex2(s[t][3] - m1);
      l[0] += p0 + p1;
      l[1] += p2 + p3;
      // The tensor cores take P and V in one 16-bit type: P goes in as its
      // upper bits and what they left over (two products), so that only the
      // output itself is rounded to 16 bits.  One rounded P cost 1.3 times the
      // output's own rounding error; the second product is hidden behind HBM.
      // Both parts are above 0, so that an infinite V stays what it is (1 % of
      // the time at most: 32 ragged sequences 24.95 -> 25.2 us).
      split(p0, p1, a[2 * t], b[2 * t]);
      split(p2, p3, a[2 * t + 1], b[2 * t + 1]);
    }
#pragma unroll
    for (int d = 0; d < D / 16; ++d) {
      uint32_t f[4];
      ldsm4_t(vb + swz<Cfg::RB>((mi & 1) * 8 + ri, d * 2 + (mi >> 1)), f);
      mma16816<BF16>(o[2 * d], a, f[0], f[1]);
      mma16816<BF16>(o[2 * d + 1], a, f[2], f[3]);
      mma16816<BF16>(o[2 * d], b, f[0], f[1]);
      mma16816<BF16>(o[2 * d + 1], b, f[2], f[3]);
    }
  }

  TKB_DEVFN void finish() {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
    }
  }
  // O to so[GT][D], (m, l) to sml[GT]
  TKB_DEVFN void put(float* so, float2* sml) const {
    const int r = lane_id() >> 2, c = lane_id() & 3;
#pragma unroll
    for (int i = 0; i < GT / 8; ++i) {
#pragma unroll
      for (int d = 0; d < D / 8; ++d)
        *reinterpret_cast<float2*>(so + (r + 8 * i) * D + d * 8 + 2 * c) = make_float2(o[d][2 * i], o[d][2 * i + 1]);
      if (c == 0) sml[r + 8 * i] = make_float2(m[i], l[i]);
    }
  }
  // the finished rows
  TKB_DEVFN void store(const DecodeParams& p, int b, int h0, int rows) const {
    const int r = lane_id() >> 2, c = lane_id() & 3;
#pragma unroll
    for (int i = 0; i < GT / 8; ++i)
      if (r + 8 * i < rows) {
        const float inv = l[i] == 0.f ? 0.f : 1.0f / (l[i] * kPUp<T>);
        T* out = static_cast<T*>(p.out) + b * p.out_stride + static_cast<long long>(h0 + r + 8 * i) * D + 2 * c;
#pragma unroll
        for (int d = 0; d < D / 8; ++d)
          *reinterpret_cast<uint32_t*>(out + d * 8) = pack2<BF16>(o[d][2 * i] * inv, o[d][2 * i + 1] * inv);
        if (c == 0) decode_lse(p, b, h0 + r + 8 * i, m[i], l[i]);
      }
  }
};

// The fp32 tile on FMA units.  Scores: 32 / TK lanes share a key, each with
// every (32 / TK)-th 16-byte chunk of its row.  Output: each lane owns D / 32
// columns.  GT: query heads the registers are laid out for.
template <int D, int GT>
struct TileFma {
  using Cfg = DecodeTile<D, 4, GT>;
  static constexpr int TK = Cfg::TK, PART = 32 / TK, CH = D / 4 / PART, E = D / 32;
  static constexpr int GROUP = GT;
  float o[GT][E], m[GT], l[GT];

  TKB_DEVFN void start(const DecodeParams& p, int b, int h0, int rows, uint8_t* extra) {
    // the unit's q, scaled, in the warp's shared memory
    float* sq = reinterpret_cast<float*>(extra);
    const float* src = static_cast<const float*>(p.q) + b * p.q_stride + static_cast<long long>(h0) * D;
    __syncwarp();
    for (int i = lane_id(); i < GT * D; i += 32) sq[i] = i < rows * D ? __ldg(src + i) * p.scale_log2 : 0.f;
    __syncwarp();
#pragma unroll
    for (int g = 0; g < GT; ++g) {
      m[g] = -INFINITY;
      l[g] = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) o[g][e] = 0.f;
    }
  }

  TKB_DEVFN void tile(const DecodeParams&, const uint8_t* buf, uint8_t* extra, int valid, int rows, float* scores,
                      long long score_stride) {
    const int lane = lane_id(), part = lane % PART;
    // neighbouring keys in a phase of eight lanes differ in the bit that the swizzle moves by 64 bytes
    const int kk = lane / PART;
    const int key = TK == 8 ? ((kk & 1) << 2) | (kk >> 1) : ((kk & 3) << 1) | ((kk >> 2) & 1) | (kk & 8);
    const float* sq = reinterpret_cast<const float*>(extra);
    float* sp = reinterpret_cast<float*>(extra + GT * D * 4);
    float4 k[CH];
#pragma unroll
    for (int i = 0; i < CH; ++i)
      k[i] = *reinterpret_cast<const float4*>(buf + swz<Cfg::RB>(key, part + PART * i));
    // all GT heads without branches, so that their chains overlap (heads past `rows` have q = 0)
    float s[GT];
#pragma unroll
    for (int g = 0; g < GT; ++g) {
      s[g] = 0.f;
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const float4 q = *reinterpret_cast<const float4*>(sq + g * D + (part + PART * i) * 4);
        s[g] = fmaf(q.x, k[i].x, s[g]);
        s[g] = fmaf(q.y, k[i].y, s[g]);
        s[g] = fmaf(q.z, k[i].z, s[g]);
        s[g] = fmaf(q.w, k[i].w, s[g]);
      }
    }
#pragma unroll
    for (int d = 1; d < PART; d <<= 1)
#pragma unroll
      for (int g = 0; g < GT; ++g) s[g] += __shfl_xor_sync(0xffffffffu, s[g], d);
    float x[GT];
#pragma unroll
    for (int g = 0; g < GT; ++g) {
      if (key >= valid) s[g] = -INFINITY;
      x[g] = s[g];
    }
    if (scores && part == 0)
#pragma unroll
      for (int g = 0; g < GT; ++g)
        if (g < rows) scores[g * score_stride + key] = s[g];
#pragma unroll
    for (int d = PART; d < 32; d <<= 1)
#pragma unroll
      for (int g = 0; g < GT; ++g) x[g] = fmaxf(x[g], __shfl_xor_sync(0xffffffffu, x[g], d));
#pragma unroll
    for (int g = 0; g < GT; ++g) {
      const float mn = fmaxf(m[g], x[g]);
      // the maximum passes over NaN: where it is still -inf, nothing but masked keys (ex2 gives 0) or NaN (and it stays NaN)
      const float keep = m[g] == -INFINITY ? 0.f : ex2(m[g] - mn), pr = ex2(s[g] - (mn == -INFINITY ? 0.f : mn));
      m[g] = mn;
      // every lane adds its own key's share: the lanes of a key carry it PART times
      l[g] = l[g] * keep + pr;
#pragma unroll
      for (int e = 0; e < E; ++e) o[g][e] *= keep;
      if (part == 0) sp[g * TK + key] = pr;
    }
    __syncwarp();
    const uint8_t* vb = buf + Cfg::HALF;
#pragma unroll
    for (int j = 0; j < TK; ++j) {
      float v[E];
      const uint8_t* at = vb + swz<Cfg::RB>(j, lane * E / 4) + (lane * E % 4) * 4;
      if constexpr (E == 4) {
        const float4 t = *reinterpret_cast<const float4*>(at);
        v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
      } else {
        const float2 t = *reinterpret_cast<const float2*>(at);
        v[0] = t.x; v[1] = t.y;
      }
#pragma unroll
      for (int g = 0; g < GT; ++g) {
        const float pr = sp[g * TK + j];
#pragma unroll
        for (int e = 0; e < E; ++e) o[g][e] = fmaf(pr, v[e], o[g][e]);
      }
    }
    __syncwarp();
  }

  TKB_DEVFN void finish() {
#pragma unroll
    for (int g = 0; g < GT; ++g) l[g] = warp_sum(l[g]) * (1.0f / PART);
  }
  TKB_DEVFN void put(float* so, float2* sml) const {
#pragma unroll
    for (int g = 0; g < GT; ++g) {
#pragma unroll
      for (int e = 0; e < E; ++e) so[g * D + lane_id() * E + e] = o[g][e];
      if (lane_id() == 0) sml[g] = make_float2(m[g], l[g]);
    }
  }
  TKB_DEVFN void store(const DecodeParams& p, int b, int h0, int rows) const {
#pragma unroll
    for (int g = 0; g < GT; ++g)
      if (g < rows) decode_store<float, E>(p, b, h0 + g, lane_id(), m[g], l[g], o[g]);
  }
};

// What a warp left of a unit that does not lie inside its run.
struct DecodePart {
  int b, u;         // sequence (-1: nothing), (kv head, query block)
  int unit0, nt;    // first tile of the unit, its number of tiles
};

template <typename T, int D, typename Tile>
__global__ void __launch_bounds__(Tile::Cfg::WARPS * 32, 1)
    paged_decode_kernel(const __grid_constant__ DecodeParams p) {
  using Cfg = typename Tile::Cfg;
  constexpr int TK = Cfg::TK, ST = Cfg::STAGES, E = D / 32, DW = Cfg::WARPS, DNT = DW * 32, GT = Tile::GROUP;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float2 s_ml[2 * DW][GT];
  __shared__ DecodePart s_part[2 * DW];
  __shared__ int3 s_at[DW];  // sequence, tokens it holds, tiles of it before the warp's first
  __shared__ int s_start[DW], s_last[2];
  const tkb_kv_cache& c = p.c;
  const int w = warp_id(), lane = lane_id(), tid = threadIdx.x, units = c.Hkv * p.qblocks;
  uint8_t* ring = smem + w * Cfg::RING;
  uint8_t* extra = smem + DW * (Cfg::RING + Cfg::HEAD) + w * Cfg::EXTRA;
  auto head_of = [&](int i) {
    return Cfg::HEAD ? reinterpret_cast<float*>(smem + DW * Cfg::RING + i * Cfg::HEAD)
                     : p.head + (static_cast<long long>(blockIdx.x) * DW + i) * GT * D;
  };

  grid_wait();
  // ---- this CTA's run of tiles, [t0, t1) of all `total` ones
  const int per = (c.B + DNT - 1) / DNT, q0 = min(c.B, tid * per), q1 = min(c.B, q0 + per);
  int mine = 0, held = 0;
  for (int b = q0; b < q1; ++b) {
    held = held_of(c, b);
    mine += max(1, (held + TK - 1) / TK) * units;
  }
  int pre = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, pre, d);
    if (lane >= d) pre += t;
  }
  if (lane == 31) s_start[w] = pre;
  if (lane < 2) s_part[2 * w + lane].b = -1;
  __syncthreads();
  int total = 0, before = pre - mine;
#pragma unroll
  for (int i = 0; i < DW; ++i) {
    if (i < w) before += s_start[i];
    total += s_start[i];
  }
  // fewer CTAs than the grid when there is not a tile for every warp
  const int ctas = min(static_cast<int>(gridDim.x), (total + DW - 1) / DW);
  if (static_cast<int>(blockIdx.x) >= ctas) return;
  auto run_of = [&](int i) { return static_cast<int>(static_cast<long long>(total) * i / ctas); };
  const int t0 = run_of(blockIdx.x), t1 = run_of(blockIdx.x + 1);
  // the thread that counted a warp's first tile says so (and no more: with the
  // divisions here too, one thread did them for all the warps in turn)
#pragma unroll 1
  for (int i = 0; i < DW; ++i) {
    const int r = t0 + (t1 - t0) * i / DW - before;
    if (r >= 0 && r < mine) s_at[i] = make_int3(q0, held, r);
  }
  __syncthreads();
  // this warp's run, [t, tw)
  int t = t0 + (t1 - t0) * w / DW;
  const int tw = t0 + (t1 - t0) * (w + 1) / DW;
  TileAt cur;
  cur.b = c.B;
  if (t < tw) {
    const int3 at = s_at[w];
    int r = at.z;
    cur.b = at.x;
    cur.n = per > 1 ? held_of(c, cur.b) : at.y;
    cur.nt = max(1, (cur.n + TK - 1) / TK);
    while (r >= cur.nt * units) {
      r -= cur.nt * units;
      ++cur.b;
      tile_seq<TK>(c, cur);
    }
    cur.u = r / cur.nt;
    cur.j = r - cur.u * cur.nt;
  }

  // ---- loads.  Lane i holds entry pbase + i of the sequence's page table, and
  // the entry 32 further: both were asked for long before they are needed.
  TileAt ld = cur;
  int lt = t, lstage = 0, valid_ring = 0, ldb = -1, pbase = 0, pages = -1, pages_next = -1;
  int pi = cur.j * TK / c.page_size, in_page = cur.j * TK - pi * c.page_size;
  auto table = [&](int i) {
    return i < c.max_pages ? __ldg(c.block_table + static_cast<long long>(ldb) * c.max_pages + i) : -1;
  };
  auto issue = [&]() {
    if (lt < tw) {
      if (ldb != ld.b || pi < pbase || pi >= pbase + 64) {
        ldb = ld.b;
        pbase = pi;
        pages = table(pbase + lane);
        pages_next = table(pbase + 32 + lane);
      } else if (pi >= pbase + 32) {
        pbase += 32;
        pages = pages_next;
        pages_next = table(pbase + 32 + lane);
      }
      int page = __shfl_sync(0xffffffffu, pages, pi - pbase);
      int valid = min(max(ld.n - ld.j * TK, 0), TK);
      if (valid == 0) {
        page = -1;
      } else if (static_cast<unsigned>(page) >= static_cast<unsigned>(c.n_pages)) {
        atomicOr(&g_device_error, ERR_BAD_INDEX);
        page = -1;
        valid = 0;
      }
      const long long off =
          page < 0 ? 0 : (page_offset(c, page, ld.u / p.qblocks) + static_cast<long long>(in_page) * D) *
                             static_cast<long long>(sizeof(T));
      const uint8_t* gk = static_cast<const uint8_t*>(c.k) + off;
      const uint8_t* gv = static_cast<const uint8_t*>(c.v) + off;
      const uint32_t dst = smem_u32(ring + lstage * 2 * Cfg::HALF);
      constexpr int CPR = Cfg::RB / 16, RPI = 32 / CPR;  // chunks per row, rows per pass of the warp
#pragma unroll
      for (int i = 0; i < TK / RPI; ++i) {
        const int r = i * RPI + lane / CPR, ch = lane % CPR;
        const int ok = r < valid ? 16 : 0;  // slots past the length are filled with zeros, not read
        const int go = ok ? r * Cfg::RB + ch * 16 : 0;
        cp_async16(dst + swz<Cfg::RB>(r, ch), gk + go, ok);
        cp_async16(dst + Cfg::HALF + swz<Cfg::RB>(r, ch), gv + go, ok);
      }
      valid_ring = (valid_ring & ~(31 << (5 * lstage))) | (valid << (5 * lstage));
      ++lt;
      in_page += TK;
      if (in_page == c.page_size) {
        in_page = 0;
        ++pi;
      }
      if (++ld.j == ld.nt) {
        ld.j = pi = in_page = 0;
        if (++ld.u == units) {
          ld.u = 0;
          ++ld.b;
          tile_seq<TK>(c, ld);
        }
      }
    }
    cp_async_commit();
    lstage = lstage + 1 == ST ? 0 : lstage + 1;
  };
#pragma unroll
  for (int i = 0; i < ST - 1; ++i) issue();

  // ---- this warp's units
  Tile tile;
  int stage = 0;
  const long long cap = static_cast<long long>(c.max_pages) * c.page_size;
  while (t < tw) {
    const int unit0 = t - cur.j, unit1 = unit0 + cur.nt, end = min(tw, unit1);
    const int g0 = (cur.u % p.qblocks) * QT, rows = min(QT, p.G - g0), h0 = (cur.u / p.qblocks) * p.G + g0;
    tile.start(p, cur.b, h0, rows, extra);
    float* scores = p.accumulate ? p.scores + (static_cast<long long>(cur.b) * p.Hq + h0) * cap : nullptr;
    const bool first = t == unit0;
    for (; t < end; ++t) {
      cp_async_wait<ST - 2>();
      __syncwarp();
      const int valid = (valid_ring >> (5 * stage)) & 31;
      const uint8_t* buf = ring + stage * 2 * Cfg::HALF;
      issue();  // into the stage that the last tile has left
      tile.tile(p, buf, extra, valid, rows, scores ? scores + static_cast<long long>(t - unit0) * TK : nullptr, cap);
      __syncwarp();
      stage = stage + 1 == ST ? 0 : stage + 1;
    }
    tile.finish();
    if (first && end == unit1) {
      tile.store(p, cur.b, h0, rows);
    } else {
      // a part: the unit goes on in the next run (kept in the ring, which no load will use again), or ended here
      const int i = 2 * w + (end < unit1 ? 1 : 0);
      if (end < unit1) cp_async_wait<0>();
      __syncwarp();
      tile.put(end < unit1 ? reinterpret_cast<float*>(ring) : head_of(w), s_ml[i]);
      if (lane == 0) s_part[i] = {cur.b, cur.u, unit0, cur.nt};
    }
    cur.j = 0;
    if (t < tw && ++cur.u == units) {
      cur.u = 0;
      ++cur.b;
      tile_seq<TK>(c, cur);
    }
  }
  __syncthreads();

  // ---- parts of the same unit meet.  Lane i looks at part i; a unit's parts
  // are neighbours.  (unit, row) pairs are dealt to the warps.
  DecodePart u;
  u.b = -1;
  u.unit0 = u.nt = u.u = 0;
  if (lane < 2 * DW) u = s_part[lane];
  const unsigned there = __ballot_sync(0xffffffffu, u.b >= 0);
  const unsigned below = there & ((1u << lane) - 1);
  const int prev0 = __shfl_sync(0xffffffffu, u.unit0, below ? 31 - __clz(below) : lane);
  const unsigned leads = __ballot_sync(0xffffffffu, u.b >= 0 && (!below || prev0 != u.unit0));
  const bool whole = u.unit0 >= t0 && u.unit0 + u.nt <= t1;
  // units that go on in other CTAs: at most two
  const unsigned opens = leads & __ballot_sync(0xffffffffu, !whole);
  int turn = w;  // pairs until this warp's next
  for (unsigned rest = leads; rest; rest &= rest - 1) {
    const int i = __ffs(rest) - 1;
    const unsigned after = rest & (rest - 1);
    // this unit's parts: from its leader up to the next one
    const unsigned group = there & ~((1u << i) - 1) & (after ? (1u << (__ffs(after) - 1)) - 1 : 0xffffffffu);
    const int ub = __shfl_sync(0xffffffffu, u.b, i), uu = __shfl_sync(0xffffffffu, u.u, i);
    const int unit0 = __shfl_sync(0xffffffffu, u.unit0, i);
    const int g0 = (uu % p.qblocks) * QT, rows = min(QT, p.G - g0), h0 = (uu / p.qblocks) * p.G + g0;
    int g = turn;
    for (; g < rows; g += DW) {
      float2 ml = make_float2(-INFINITY, 0.f);
      if (group >> lane & 1) ml = s_ml[lane][g];
      const float M = warp_max(ml.x);
      const float f = ml.x == M ? 1.f : ex2(ml.x - M);
      const float L = warp_sum(f * ml.y);
      float acc[E];
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = 0.f;
      for (unsigned m = group; m; m &= m - 1) {
        const int k = __ffs(m) - 1;
        const float fk = __shfl_sync(0xffffffffu, f, k);
        const float* so = (k & 1 ? reinterpret_cast<const float*>(smem + (k >> 1) * Cfg::RING) : head_of(k >> 1)) + g * D + lane * E;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = fmaf(fk, so[e], acc[e]);
      }
      if (!(opens >> i & 1)) {
        decode_store<T, E>(p, ub, h0 + g, lane, M, L, acc);
      } else {
        float* at = p.part + (static_cast<long long>(2 * blockIdx.x + (t0 >= unit0 ? 0 : 1)) * QT + g) * (D + 2);
#pragma unroll
        for (int e = 0; e < E; ++e) at[lane * E + e] = acc[e];
        if (lane == 0) {
          at[D] = M;
          at[D + 1] = L;
        }
      }
    }
    turn = g - rows;
  }
  if (!opens) return;

  // ---- the CTA that ends last joins the unit's parts, in the order of the runs
  __syncthreads();
  const int left = __popc(opens), o0 = __ffs(opens) - 1, o1 = 31 - __clz(opens);
  auto first_cta = [&](int unit0) { return static_cast<int>((static_cast<long long>(unit0 + 1) * ctas - 1) / total); };
  if (w == 0 && (opens >> lane & 1)) {
    const int c0 = first_cta(u.unit0), c1 = first_cta(u.unit0 + u.nt - 1);
    __threadfence();
    int* counter = &p.counters[c0];
    const bool last = atomicAdd(counter, 1) == c1 - c0;
    s_last[lane == o0 ? 0 : 1] = last;
    if (last) *counter = 0;  // for the next call
    __threadfence();
  }
  __syncthreads();
  for (int x = 0; x < left; ++x) {
    if (!s_last[x]) continue;
    const int i0 = x ? o1 : o0;
    const int ub = __shfl_sync(0xffffffffu, u.b, i0), uu = __shfl_sync(0xffffffffu, u.u, i0);
    const int unit0 = __shfl_sync(0xffffffffu, u.unit0, i0), nt = __shfl_sync(0xffffffffu, u.nt, i0);
    const int g0 = (uu % p.qblocks) * QT, rows = min(QT, p.G - g0), h0 = (uu / p.qblocks) * p.G + g0;
    const int c0 = first_cta(unit0), c1 = first_cta(unit0 + nt - 1);
    for (int g = w; g < rows; g += DW) {
      // CTA i's part is its first when its run starts inside the unit, else its second: only c0 may start before
      const long long stride = 2ll * QT * (D + 2);
      const float* part0 = p.part + (static_cast<long long>(2 * c0 + (run_of(c0) >= unit0 ? 0 : 1)) * QT + g) * (D + 2);
      const float* part1 = p.part + (static_cast<long long>(2 * c0) * QT + g) * (D + 2);
      auto part = [&](int i) { return i == c0 ? part0 : part1 + (i - c0) * stride; };
      // four parts' loads at a time, none waiting for another's
      float M = -INFINITY, L = 0.f, acc[E];
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = 0.f;
      for (int i = c0; i <= c1; i += 4) {
        float m[4], l[4], v[4][E];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          m[k] = -INFINITY;
          l[k] = 0.f;
#pragma unroll
          for (int e = 0; e < E; ++e) v[k][e] = 0.f;
          if (i + k <= c1) {
            const float* at = part(i + k);
            m[k] = __ldcg(at + D);
            l[k] = __ldcg(at + D + 1);
#pragma unroll
            for (int e = 0; e < E; ++e) v[k][e] = __ldcg(at + lane * E + e);
          }
        }
        const float Mn = fmaxf(fmaxf(fmaxf(M, m[0]), fmaxf(m[1], m[2])), m[3]);
        const float f = M == Mn ? 1.f : ex2(M - Mn);
        M = Mn;
        L *= f;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] *= f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float fk = m[k] == M ? 1.f : ex2(m[k] - M);
          L = fmaf(fk, l[k], L);
#pragma unroll
          for (int e = 0; e < E; ++e) acc[e] = fmaf(fk, v[k][e], acc[e]);
        }
      }
      decode_store<T, E>(p, ub, h0 + g, lane, M, L, acc);
    }
  }
}

// weight[slot] += sum over the group's query heads of exp(s - lse): the second
// pass of `accumulate`, over the scores the first one kept (4 G bytes per key
// and kv head beside the 2 D values of K and V).  A thread takes four slots:
// pages are multiples of 16, so one page holds them.
__global__ void __launch_bounds__(256) paged_weight_kernel(const __grid_constant__ DecodeParams p) {
  const tkb_kv_cache& c = p.c;
  const int b = blockIdx.y / c.Hkv, h = blockIdx.y % c.Hkv, j = (blockIdx.x * 256 + threadIdx.x) * 4;
  grid_wait();
  const int n = held_of(c, b);
  if (j >= n) return;
  const int pg = j / c.page_size, page = page_of(c, b, pg);
  if (page < 0) return;
  const long long cap = static_cast<long long>(c.max_pages) * c.page_size;
  const float* s = p.scores + (static_cast<long long>(b) * p.Hq + h * p.G) * cap + j;
  const float* lse2 = p.lse2 + static_cast<long long>(b) * p.Hq + h * p.G;
  float4* at = reinterpret_cast<float4*>(c.weight + meta_offset(c, page, h) + (j - pg * c.page_size));
  float4 sum = *at;
#pragma unroll 8
  for (int g = 0; g < p.G; ++g) {
    const float4 x = __ldcs(reinterpret_cast<const float4*>(s + g * cap));
    const float l = lse2[g];
    sum.x += ex2(x.x - l);
    if (j + 1 < n) sum.y += ex2(x.y - l);
    if (j + 2 < n) sum.z += ex2(x.z - l);
    if (j + 3 < n) sum.w += ex2(x.w - l);
  }
  *at = sum;
}

constexpr int kDecodeGrid = 148;  // one CTA per SM

// Workspace: counters, partial results, then (accumulate) lse2 and scores.  The
// counters alone keep a state between calls; they lie first and are as many for
// every shape, since one call's data over another's counters would lose joins.
struct DecodeWs {
  size_t counters, part, head, lse2, scores, bytes;
};
static DecodeWs decode_ws(const tkb_kv_cache& c, int Hq, int accumulate) {
  auto up = [](size_t x) { return (x + 255) & ~size_t(255); };
  const int G = Hq / c.Hkv;
  DecodeWs w;
  w.counters = 0;
  w.part = up(kDecodeGrid * 4);
  w.head = w.part + up(static_cast<size_t>(2) * kDecodeGrid * QT * (c.D + 2) * 4);
  // the 16-row tiles (paged_decode_d) keep their first parts here
  w.lse2 = w.head + (G > 8 ? up(static_cast<size_t>(kDecodeGrid) * 16 * QT * c.D * 4) : 0);
  w.scores = w.lse2 + (accumulate ? up(static_cast<size_t>(c.B) * Hq * 4) : 0);
  w.bytes = w.scores + (accumulate ? up(static_cast<size_t>(c.B) * Hq * c.max_pages * c.page_size * 4) : 0);
  return w;
}

template <typename T, int D, typename Tile>
static cudaError_t paged_decode_launch(const DecodeParams& p, cudaStream_t st) {
  using Cfg = typename Tile::Cfg;
  constexpr int W = Cfg::WARPS;
  auto k = paged_decode_kernel<T, D, Tile>;
  cudaError_t e = allow_smem<paged_decode_kernel<T, D, Tile>>(Cfg::SMEM);
  if (e != cudaSuccess) return e;
  const long long most = static_cast<long long>(p.c.B) * p.c.Hkv * p.qblocks * (p.c.max_pages * p.c.page_size / Cfg::TK);
  const int grid = static_cast<int>(most < kDecodeGrid * W ? (most + W - 1) / W : kDecodeGrid);
  return launch_early(k, dim3(grid), W * 32, Cfg::SMEM, st, p);
}

// Rows of a tile by the query heads per kv head.  16-bit: 8 or 16, since parts
// of 16 rows have no room in shared memory beside three stages of loads.
// fp32: the registers and shared memory of q grow with them, and heads that are
// not there cost as much as those that are; 8 sequences of 3-4 k tokens, 4 kv
// heads of 128 (floor 18 us): 1 head 32 us, 4 heads 35 (with one branch per
// head, 41), 8 heads 52 (in the 16-row tile, with branches, 81), 16 heads 91.
template <typename T, int D>
static cudaError_t paged_decode_d(const DecodeParams& p, cudaStream_t st) {
  if constexpr (sizeof(T) == 2) {
    if (p.G <= 8) return paged_decode_launch<T, D, TileMma<T, D, 8>>(p, st);
    return paged_decode_launch<T, D, TileMma<T, D, 16>>(p, st);
  } else {
    if (p.G == 1) return paged_decode_launch<T, D, TileFma<D, 1>>(p, st);
    if (p.G <= 4) return paged_decode_launch<T, D, TileFma<D, 4>>(p, st);
    if (p.G <= 8) return paged_decode_launch<T, D, TileFma<D, 8>>(p, st);
    return paged_decode_launch<T, D, TileFma<D, 16>>(p, st);
  }
}

template <typename T>
static cudaError_t paged_decode_t(const DecodeParams& p, cudaStream_t st) {
  cudaError_t e = p.c.D == 64 ? paged_decode_d<T, 64>(p, st) : paged_decode_d<T, 128>(p, st);
  if (e == cudaSuccess && p.accumulate) {
    const long long cap = static_cast<long long>(p.c.max_pages) * p.c.page_size;
    e = launch_early(paged_weight_kernel, dim3(static_cast<unsigned>((cap + 1023) / 1024), p.c.B * p.c.Hkv), 256, 0, st, p);
  }
  return e;
}

// ============================================================ eviction
// Per (sequence, kv head): the budget-th largest key by a radix search over
// counts (11, 11 and 10 bits), then the freed slots below the budget and the kept tokens above it, both in
// ascending order, then the moves.  Reads 8 bytes per slot; the moves (read
// and written once) are what HBM is busy with, so several CTAs share a unit
// when there are few units.  They form a cluster: each finds the same cut from
// the same keys (held in shared memory, or in the workspace when a sequence
// has room for more than kEvictSmemKeys), and the barrier between the reading of the keys and
// the moves keeps a fast one from changing what a slow one still reads.
// Measured: 4 sequences of 12-16 k tokens to 2048, 8 heads of 128, f16 (63 MB
// with the moves): 35 us, of which keys 4, cut 10, lists 6, moves 10; 32
// sequences of 1000-1088 to 1024: 10 us.
constexpr int kEvictSmemKeys = 49152;

struct EvictParams {
  tkb_kv_cache c;
  const int32_t* seen;
  uint2* lists;     // per unit: `cap` destinations (page, slot in page), then `cap` sources
  uint32_t* keys;   // per CTA: room for every slot, or null (shared memory)
  int budget, recent, sinks, cap, split;
};

// Floats as unsigned numbers of the same order (-0 as +0, NaN below -inf).
TKB_DEVFN uint32_t order_key(float x) {
  if (x != x) return 0u;
  const uint32_t u = __float_as_uint(x + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Exclusive prefix over the warps of a warp-uniform count.
template <int THREADS>
TKB_DEVFN int evict_prefix(int v, int* sh, int turn, int& total) {
  if (lane_id() == 0) sh[turn * (THREADS / 32) + warp_id()] = v;
  __syncthreads();
  const int x = lane_id() < THREADS / 32 ? sh[turn * (THREADS / 32) + lane_id()] : 0;
  total = __reduce_add_sync(0xffffffffu, x);
  return __reduce_add_sync(0xffffffffu, lane_id() < warp_id() ? x : 0);
}

template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS) kv_evict_kernel(const __grid_constant__ EvictParams p) {
  constexpr int W = THREADS / 32;
  extern __shared__ __align__(16) uint32_t s_keys[];
  __shared__ int sh[2 * W], hist[2048], s_cut[3];
  const tkb_kv_cache& c = p.c;
  const int unit = blockIdx.x / p.split, rank = blockIdx.x % p.split;
  const int b = unit / c.Hkv, h = unit % c.Hkv, tid = threadIdx.x, w = warp_id(), lane = lane_id();
  grid_wait();
  const int n = held_of(c, b), ps = c.page_size;
  if (n <= p.budget) return;  // the whole cluster
  uint32_t* keys = p.keys ? p.keys + static_cast<long long>(blockIdx.x) * c.max_pages * ps : s_keys;

  // ---- keys: protected tokens above all others
  const int newest = p.seen[b] - p.recent;
  const bool by_pos = p.recent > 0 || p.sinks > 0;
  const int32_t* table = c.block_table + static_cast<long long>(b) * c.max_pages;
  // four slots a thread: pages are multiples of 16, so one page holds them
#pragma unroll 4
  for (int j = 4 * tid; j < n; j += 4 * THREADS) {
    const int pg = j / ps, page = __ldg(table + pg);
    uint4 k = make_uint4(0u, 0u, 0u, 0u);
    if (static_cast<unsigned>(page) < static_cast<unsigned>(c.n_pages)) {
      const long long at = meta_offset(c, page, h) + (j - pg * ps);
      const float4 x = *reinterpret_cast<const float4*>(c.weight + at);
      k = make_uint4(order_key(x.x), order_key(x.y), order_key(x.z), order_key(x.w));
      if (by_pos) {
        const int4 pos = *reinterpret_cast<const int4*>(c.pos + at);
        if (pos.x >= newest || pos.x < p.sinks) k.x = 0xFFFFFFFFu;
        if (pos.y >= newest || pos.y < p.sinks) k.y = 0xFFFFFFFFu;
        if (pos.z >= newest || pos.z < p.sinks) k.z = 0xFFFFFFFFu;
        if (pos.w >= newest || pos.w < p.sinks) k.w = 0xFFFFFFFFu;
      }
    } else {
      atomicOr(&g_device_error, ERR_BAD_INDEX);
    }
    *reinterpret_cast<uint4*>(keys + j) = k;  // the key area holds whole pages
  }

  // ---- the cut: the largest key that at least `budget` tokens reach.  Weights
  // differ in their first 11 bits (sign, exponent, two bits) enough to spread
  // the first histogram; a warp whose keys agree adds once.
  uint32_t lo = 0;
  int need = p.budget;  // of the tokens that share lo's bits so far
  int in_bin = 0;
#pragma unroll 1
  for (int level = 0; level < 3; ++level) {
    const int shift = level == 0 ? 21 : level == 1 ? 10 : 0, bits = level == 2 ? 10 : 11, bins = 1 << bits;
    for (int i = tid; i < bins; i += THREADS) hist[i] = 0;
    __syncthreads();
    for (int j0 = 0; j0 < n; j0 += 4 * THREADS) {
      const int j = j0 + 4 * tid;
      const uint4 q = j < n ? *reinterpret_cast<const uint4*>(keys + j) : make_uint4(0u, 0u, 0u, 0u);
      const uint32_t k4[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool in = j + e < n && (level == 0 || ((k4[e] ^ lo) >> (shift + bits)) == 0);
        const int bin = static_cast<int>((k4[e] >> shift) & (bins - 1));
        const unsigned m = __ballot_sync(0xffffffffu, in);
        if (!m) continue;
        const int lead = __ffs(m) - 1, first = __shfl_sync(0xffffffffu, bin, lead);
        if (__all_sync(0xffffffffu, !in || bin == first)) {
          if (lane == lead) atomicAdd(&hist[first], __popc(m));
        } else if (in) {
          atomicAdd(&hist[bin], 1);
        }
      }
    }
    __syncthreads();
    // thread t: the bins from the top, `run` at a time
    const int run = bins / THREADS;
    int sum = 0;
    for (int i = 0; i < run; ++i) sum += hist[bins - 1 - tid * run - i];
    int upto = sum;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += o;
    }
    if (lane == 31) sh[w] = upto;
    __syncthreads();
    const int x = lane < W ? sh[lane] : 0;
    upto += __reduce_add_sync(0xffffffffu, lane < w ? x : 0);
    if (upto >= need && upto - sum < need) {
      int above = upto - sum, bin = bins - 1 - tid * run;
      while (above + hist[bin] < need) above += hist[bin--];
      s_cut[0] = bin;
      s_cut[1] = need - above;
      s_cut[2] = hist[bin];
    }
    __syncthreads();
    lo |= static_cast<uint32_t>(s_cut[0]) << shift;
    need = s_cut[1];
    in_bin = s_cut[2];
  }
  // kept: the keys above lo, and of those equal to it the first `need`
  const int chunk = (n + 4 * THREADS - 1) / (4 * THREADS) * 128, j0 = min(n, w * chunk), j1 = min(n, j0 + chunk);
  const bool some = need < in_bin;  // not all tokens of key lo stay: their order counts
  int tie_base = 0;
  if (some) {
    int ties = 0, total;
    for (int j = j0 + lane; j < j1; j += 32) ties += keys[j] == lo;
    __syncthreads();
    tie_base = evict_prefix<THREADS>(__reduce_add_sync(0xffffffffu, ties), sh, 1, total);
    __syncthreads();
  }
  // `f(j, hole, mover)` for the warp's slots in order, four a lane: bit e of
  // the masks stands for slot j + e
  auto walk = [&](auto f) {
    int rank_base = tie_base;
    for (int jj = j0; jj < j1; jj += 128) {
      const int j = jj + 4 * lane;
      const uint4 q = j < j1 ? *reinterpret_cast<const uint4*>(keys + j) : make_uint4(0u, 0u, 0u, 0u);
      const uint32_t k4[4] = {q.x, q.y, q.z, q.w};
      unsigned in = 0, kept = 0, tie = 0, low = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (j + e < j1) in |= 1u << e;
        if (j + e < p.budget) low |= 1u << e;
        if (k4[e] > lo) kept |= 1u << e;
        if (k4[e] == lo) tie |= 1u << e;
      }
      kept &= in;
      tie &= in;
      if (some) {
        int upto = __popc(tie);
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const int o = __shfl_up_sync(0xffffffffu, upto, d);
          if (lane >= d) upto += o;
        }
        int rank = rank_base + upto - __popc(tie);
        rank_base += __shfl_sync(0xffffffffu, upto, 31);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (tie >> e & 1) {
            if (rank >= need) tie &= ~(1u << e);
            ++rank;
          }
      }
      kept |= tie;
      f(j, in & ~kept & low, kept & ~low);
    }
  };
  int holes = 0, movers = 0, total;
  walk([&](int, unsigned hole, unsigned mover) {
    holes += __popc(hole);
    movers += __popc(mover);
  });
  int hole_at = evict_prefix<THREADS>(__reduce_add_sync(0xffffffffu, holes), sh, 0, total);
  int mover_at = evict_prefix<THREADS>(__reduce_add_sync(0xffffffffu, movers), sh, 1, total);  // as many as holes
  // this CTA's share of the moves
  const int m0 = static_cast<int>(static_cast<long long>(total) * rank / p.split);
  const int m1 = static_cast<int>(static_cast<long long>(total) * (rank + 1) / p.split);
  uint2* to = p.lists + static_cast<long long>(unit) * 2 * p.cap;
  uint2* from = to + p.cap;
  walk([&](int j, unsigned hole, unsigned mover) {
    const int mine = __popc(hole) | __popc(mover) << 16;
    int upto = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += o;
    }
    const int all = __shfl_sync(0xffffffffu, upto, 31);
    upto -= mine;
    if (mine) {
      const int pg = j / ps;  // one page holds the four slots
      const uint32_t page = __ldg(table + pg);
      int at = hole_at + (upto & 0xFFFF);
      for (; hole; hole &= hole - 1, ++at)
        if (at >= m0 && at < m1) to[at] = make_uint2(page, j + __ffs(hole) - 1 - pg * ps);
      at = mover_at + (upto >> 16);
      for (; mover; mover &= mover - 1, ++at)
        if (at >= m0 && at < m1) from[at] = make_uint2(page, j + __ffs(mover) - 1 - pg * ps);
    }
    hole_at += all & 0xFFFF;
    mover_at += all >> 16;
  });
  __syncthreads();
  if (p.split > 1) cluster_sync();  // every CTA of the unit has read its keys

  // ---- the moves
  for (int i = m0 + tid; i < m1; i += THREADS) {
    const uint2 d = to[i], s = from[i];
    if (d.x >= static_cast<unsigned>(c.n_pages) || s.x >= static_cast<unsigned>(c.n_pages)) continue;
    const long long dm = meta_offset(c, d.x, h) + d.y, sm = meta_offset(c, s.x, h) + s.y;
    c.pos[dm] = c.pos[sm];
    c.weight[dm] = c.weight[sm];
  }
  const int vecs = c.D * static_cast<int>(sizeof(T)) / 16, per = 2 * vecs;  // a power of two each
  const int shift = 31 - __clz(per);
  const long long items = static_cast<long long>(m1 - m0) << shift;
  constexpr int U = 4;
  for (long long i0 = tid; i0 < items; i0 += U * THREADS) {
    uint4 v[U];
    uint4* dst[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const long long i = i0 + k * THREADS;
      dst[k] = nullptr;
      if (i < items) {
        const int m = m0 + static_cast<int>(i >> shift), o = static_cast<int>(i) & (per - 1);
        const uint2 d = to[m], s = from[m];
        if (d.x < static_cast<unsigned>(c.n_pages) && s.x < static_cast<unsigned>(c.n_pages)) {
          T* pool = static_cast<T*>(o < vecs ? c.k : c.v);
          const int ch = o & (vecs - 1);
          dst[k] = reinterpret_cast<uint4*>(pool + page_offset(c, d.x, h) + static_cast<long long>(d.y) * c.D) + ch;
          v[k] = reinterpret_cast<const uint4*>(pool + page_offset(c, s.x, h) + static_cast<long long>(s.y) * c.D)[ch];
        }
      }
    }
#pragma unroll
    for (int k = 0; k < U; ++k)
      if (dst[k]) *dst[k] = v[k];
  }
}

// CTAs per (sequence, kv head): a power of two up to 8 (the portable cluster
// size) that gives every SM about one.
static int evict_split(const tkb_kv_cache& c) {
  int s = 1;
  while (s < 8 && static_cast<long long>(c.B) * c.Hkv * s * 2 <= 148) s *= 2;
  return s;
}
struct EvictWs {
  size_t keys, bytes;
  int cap;
};
static EvictWs evict_ws(const tkb_kv_cache& c) {
  const size_t slots = static_cast<size_t>(c.max_pages) * c.page_size, units = static_cast<size_t>(c.B) * c.Hkv;
  EvictWs w;
  w.cap = static_cast<int>(slots / 2);  // moves: at most half of the slots
  w.keys = (units * 2 * w.cap * sizeof(uint2) + 255) & ~size_t(255);
  w.bytes = w.keys + (slots > kEvictSmemKeys ? units * evict_split(c) * slots * 4 : 0);
  return w;
}

template <typename T, int THREADS>
static cudaError_t kv_evict_launch(EvictParams p, cudaStream_t st) {
  const long long slots = static_cast<long long>(p.c.max_pages) * p.c.page_size;
  p.split = evict_split(p.c);
  const size_t smem = p.keys ? 0 : static_cast<size_t>(slots) * 4;
  cudaError_t e = allow_smem<kv_evict_kernel<T, THREADS>>(kEvictSmemKeys * 4);
  if (e != cudaSuccess) return e;
  return launch_early(kv_evict_kernel<T, THREADS>, dim3(static_cast<unsigned>(p.c.B) * p.c.Hkv * p.split), THREADS, smem,
                      st, p, p.split);
}

template <typename T>
static cudaError_t kv_evict_t(const EvictParams& p, cudaStream_t st) {
  return static_cast<long long>(p.c.max_pages) * p.c.page_size <= 4096 ? kv_evict_launch<T, 256>(p, st)
                                                                      : kv_evict_launch<T, 1024>(p, st);
}

}  // namespace tkb
