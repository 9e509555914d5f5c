// lora.cu -- low-rank adapters of many requests beside a shared projection:
// out = y + scale (x A) B with each row's own adapter.
//
// 4 R FLOP a value of x or y read: HBM bounds it for prompts (x, y and out move
// once, the adapters stay in L2), the chain of launches for single tokens.  The
// plan sorts the rows by adapter and cuts them into tiles of one adapter each
// (16 rows, or 64 where the adapters have that many), so that an adapter is
// read once a tile and its products run on m16n8k16 instructions.  Tiles of 64
// rows, and fp32, take two kernels: t = x A in fp32, cut over K into the CTAs of a cluster, which sum
// their parts in order through their shared memories; then out, cut over the
// columns.  t goes into the second product as two 16-bit values, the rounding
// and the rest, so that only out is rounded.  Tiles of 16 rows, where launches
// and first loads are what takes time, take one: the cluster that has summed t
// goes on with the columns of out.
//
// Measured, the three projections of a layer with their plan: 12.4 k rows, 8
// adapters of rank 16 (1.01 GB): 204 us, 0.76 of HBM; 64 single tokens, 16
// adapters: 27 us, four launches of 6-7; 1.6 k rows, 64 adapters of rank 64, 4096 x
// 4096: 37 us.  A block a row took 3369, 145 and 2057 us.
#include "tkb_common.cuh"
#include "../../include/tkm_b200.h"

namespace tkb {

// ============================================================ the plan
// Layout: number of tiles (256 bytes), the tiles, then the tiles' rows, tm entries each.
struct LoraTile {
  int adapter, at, count, unused;  // -1: rows without one; first sorted place, rows
};
struct LoraPlanAt {
  int tm, tiles;                   // rows per tile, tiles at most
  size_t rows, bytes;              // offset of the rows
};
static LoraPlanAt lora_plan_at(int B, int rows, int n_adapters) {
  LoraPlanAt a;
  const long long groups = n_adapters < B ? n_adapters + 1ll : B;
  // Tiles of 64 rows read an adapter a quarter as often; where adapters have few rows, most of such a tile is empty.  16 and
  // 64 rows: 1.6 k rows of 33 adapters of rank 64 73 and 37 us, 12.4 k rows of 8 315 and 204, 548 of 16 (rank 16) 11.4 and
  // 13.5, 64 of 16 27 and 37.
  a.tm = rows >= 32 * groups ? 64 : 16;
  a.tiles = static_cast<int>(rows / a.tm + (groups < rows ? groups : rows));
  a.rows = 256 + static_cast<size_t>(a.tiles) * sizeof(LoraTile);
  a.bytes = (a.rows + static_cast<size_t>(a.tiles) * a.tm * 4 + 255) & ~size_t(255);
  return a;
}

struct LoraPlanParams {
  const int32_t* adapter;
  const int32_t* row_start;
  int* n_tiles;
  LoraTile* tiles;
  int32_t* row_of;
  int B, rows, n_adapters, tm, sorted;  // sorted: power of two >= B
};
constexpr int kLoraPlanRows = 1024;     // entries of row_of per CTA: its sort is done again by each

// Every CTA sorts the sequences by adapter in shared memory, up to 256 of them
// by counting the smaller ones of each, more by a bitonic network; the sums over the
// sorted ones give places, groups of one adapter and tiles; then it writes its
// share of the tiles and rows.
template <int THREADS, int SEQS>
__global__ void __launch_bounds__(THREADS) lora_plan_kernel(const __grid_constant__ LoraPlanParams p) {
  extern __shared__ unsigned long long s_key[];           // [sorted] adapter + 1, sequence
  const int tid = threadIdx.x, n = p.sorted;
  int2* s_rows = reinterpret_cast<int2*>(s_key + n);      // [sorted] first row and number, by sequence
  int* s_pos = reinterpret_cast<int*>(s_rows + n);        // [sorted + 1] first sorted place
  int* s_group = s_pos + n + 1;                           // [sorted + 1] first sorted sequence of each group
  int* s_tile = s_group + n + 1;                          // [sorted + 1] its first tile
  __shared__ unsigned long long s_warp[32];
  grid_wait();
  grid_go();
  for (int b = tid; b < n; b += THREADS) {
    unsigned long long key = ~0ull << 16 | b;             // behind all others, and no two alike
    if (b < p.B) {
      int2 r;
      int a = p.adapter[b];
      chunk_rows(p.row_start, p.rows, b, r.x, r.y);
      if (a < -1 || a >= p.n_adapters) {
        atomicOr(&g_device_error, ERR_BAD_INDEX);
        a = -1;
      }
      if (r.y) key = static_cast<unsigned long long>(a + 1) << 32 | static_cast<unsigned>(b);
      s_rows[b] = r;
    }
    s_key[b] = key;
  }
  __syncthreads();
  if constexpr (SEQS == 1) {
    const unsigned long long key = tid < n ? s_key[tid] : 0;
    int rank = 0;
    if (tid < n)
      for (int i = 0; i < n; ++i) rank += s_key[i] < key;
    __syncthreads();
    if (tid < n) s_key[rank] = key;
    __syncthreads();
  } else {
    for (int size = 2; size <= n; size <<= 1)
      for (int stride = size >> 1; stride; stride >>= 1) {
        for (int i = tid; i < n / 2; i += THREADS) {
          const int lo = (i / stride) * 2 * stride + i % stride, hi = lo + stride;
          const unsigned long long a = s_key[lo], b = s_key[hi];
          if ((a > b) == !(lo & size)) {
            s_key[lo] = b;
            s_key[hi] = a;
          }
        }
        __syncthreads();
      }
  }
  auto holds = [&](int k) { return k < n && s_key[k] >> 48 != 0xffff; };
  auto seq_of = [&](int k) { return static_cast<int>(s_key[k] & 0xffffffffu); };
  int count[SEQS], lead[SEQS], sum = 0, leads = 0;
#pragma unroll
  for (int i = 0; i < SEQS; ++i) {
    const int k = tid * SEQS + i;
    count[i] = lead[i] = 0;
    if (!holds(k)) continue;
    count[i] = s_rows[seq_of(k)].y;
    lead[i] = k == 0 || s_key[k] >> 32 != s_key[k - 1] >> 32;
    sum += count[i];
    leads += lead[i];
  }
  // rows in the upper half: sequences that share rows can have 4096 times as many as there are
  unsigned long long all;
  const unsigned long long before = block_scan<THREADS>(static_cast<unsigned long long>(sum) << 16 | leads, s_warp, all);
  const int groups = static_cast<int>(all & 0xffff);
  const bool over = all >> 16 > static_cast<unsigned>(p.rows);
  const int total = over ? p.rows : static_cast<int>(all >> 16);
  if (over && tid == 0) atomicOr(&g_device_error, ERR_BAD_INDEX);  // those that do not fit are left out
  long long at = static_cast<long long>(before >> 16);
  int g = static_cast<int>(before & 0xffff);
#pragma unroll
  for (int i = 0; i < SEQS; ++i) {
    const int k = tid * SEQS + i;
    if (k >= n) break;
    s_pos[k] = static_cast<int>(min(at, static_cast<long long>(total)));
    if (lead[i]) s_group[g++] = k;
    at += count[i];
  }
  if (tid == 0) s_pos[n] = total;
  __syncthreads();
  auto group_start = [&](int i) { return i < groups ? s_pos[s_group[i]] : total; };
  int tiles[SEQS], mine = 0;
#pragma unroll
  for (int i = 0; i < SEQS; ++i) {
    const int k = tid * SEQS + i;
    tiles[i] = k < groups ? (group_start(k + 1) - group_start(k) + p.tm - 1) / p.tm : 0;
    mine += tiles[i];
  }
  int t = static_cast<int>(block_scan<THREADS>(static_cast<unsigned long long>(mine), s_warp, all));
  const int n_tiles = static_cast<int>(all);
#pragma unroll
  for (int i = 0; i < SEQS; ++i) {
    const int k = tid * SEQS + i;
    if (k < groups) s_tile[k] = t;
    t += tiles[i];
  }
  if (tid == 0 && blockIdx.x == 0) *p.n_tiles = n_tiles;
  __syncthreads();
  auto last_from = [](const int* from, int m, int x) {  // last of m ascending values that is x or less
    int lo = 0, hi = m - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (from[mid] <= x) lo = mid;
      else hi = mid - 1;
    }
    return lo;
  };
  const int e0 = blockIdx.x * kLoraPlanRows, e1 = min(e0 + kLoraPlanRows, n_tiles * p.tm);
  for (int e = e0 + tid; e < e1; e += THREADS) {
    const int i = e / p.tm, r = e - i * p.tm, grp = last_from(s_tile, groups, i);
    const int place = group_start(grp) + (i - s_tile[grp]) * p.tm, rows = min(p.tm, group_start(grp + 1) - place);
    if (r == 0) {
      LoraTile tile;
      tile.adapter = static_cast<int>(s_key[s_group[grp]] >> 32) - 1;
      tile.at = place;
      tile.count = rows;
      tile.unused = 0;
      p.tiles[i] = tile;
    }
    const int x = place + min(r, rows - 1);  // entries behind the tile's rows repeat the last
    const int k = last_from(s_pos, n, x);    // sequences behind the rows start at `total`
    p.row_of[e] = s_rows[seq_of(k)].x + x - s_pos[k];
  }
}

static cudaError_t lora_plan(LoraPlanParams p, int entries, cudaStream_t st) {
  p.sorted = 2;
  while (p.sorted < p.B) p.sorted *= 2;
  const size_t smem = p.sorted * 16 + (p.sorted + 1) * 3 * sizeof(int);
  const dim3 grid((entries + kLoraPlanRows - 1) / kLoraPlanRows);
  if (p.B <= 256) return launch_early(lora_plan_kernel<256, 1>, grid, 256, smem, st, p);
  const cudaError_t e = allow_smem<lora_plan_kernel<1024, 4>>(4096 * 28 + 16);
  return e != cudaSuccess ? e : launch_early(lora_plan_kernel<1024, 4>, grid, 1024, smem, st, p);
}

// ============================================================ the products
struct LoraParams {
  const int* n_tiles;
  const LoraTile* tiles;
  const int32_t* row_of;
  const void *x, *a, *b, *y;
  void* out;
  const float* scale;
  float* t;                // [rows][RP] by sorted place
  long long x_stride, y_stride, out_stride;
  int rows, K, N, R;
  int splits, k_per;       // parts of K, the CTAs of a cluster, and columns of each (a multiple of a chunk)
  int chunks;              // chunks of columns per CTA of the second kernel
};
constexpr int kLoraThreads = 128;

// Byte offset of 16-byte piece `ch` of row r in a tile of RB-byte rows, so that
// eight rows' equal pieces (ldmatrix) lie in different banks.
template <int RB>
TKB_DEVFN int lora_swz(int r, int ch) {
  return r * RB + ((ch ^ (RB == 32 ? r >> 2 & 1 : r & 7)) << 4);
}

// The parts of a tile of t, [count][RP] floats in each CTA's shared memory at
// the same place, summed in the order of the cluster's ranks; each CTA writes its share.
TKB_DEVFN void lora_meet(const float* mine, float* out, int values, int ctas) {
  if (ctas > 1) cluster_sync();
  else __syncthreads();
  const uint32_t here = smem_u32(mine);
  const int rank = blockIdx.x;  // the grid's first dimension is the cluster
  for (int i = (rank * kLoraThreads + threadIdx.x) * 4; i < values; i += ctas * kLoraThreads * 4) {
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int c = 0; c < ctas; ++c) {
      float4 v;
      if (ctas == 1) v = *reinterpret_cast<const float4*>(mine + i);
      else
        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                     : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(mapa_shared(here + i * 4, c)) : "memory");
      sum.x += v.x;
      sum.y += v.y;
      sum.z += v.z;
      sum.w += v.w;
    }
    *reinterpret_cast<float4*>(out + i) = sum;
  }
  if (ctas > 1) cluster_sync();  // the others have read this CTA's part
}

// t = x A over one part of K.  A warp holds 16 rows (of tiles of 16 rows, in
// lora_one_kernel, each has a quarter of every chunk of K instead).
template <typename T, int RP, int TM>
struct LoraDown {
  static constexpr int KC = 64, ST = 3;                  // columns of K per chunk, chunks in flight
  static constexpr int XB = TM * KC * 2, AB = KC * RP * 2, STAGE = XB + AB;
  static constexpr int SUM = (TM == 16 ? 5 : 4) * 16 * RP * 4;  // the warps' quarters and their sum, or the tile
  static constexpr int SMEM = ST * STAGE > SUM ? ST * STAGE : SUM;
};
template <typename T, int RP>
__global__ void __launch_bounds__(kLoraThreads) lora_down_kernel(const __grid_constant__ LoraParams p) {
  constexpr int TM = 64;
  using C = LoraDown<T, RP, TM>;
  constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
  extern __shared__ __align__(128) uint8_t s_ring[];
  __shared__ int s_row[TM];
  grid_wait();
  grid_go();
  const int n_tiles = *p.n_tiles;
  const LoraTile tile = p.tiles[blockIdx.y];  // read beside the number: behind it lies what an earlier plan left
  if (threadIdx.x < TM) s_row[threadIdx.x] = p.row_of[blockIdx.y * TM + threadIdx.x];
  if (static_cast<int>(blockIdx.y) >= n_tiles || tile.adapter < 0) return;
  const int tid = threadIdx.x, lane = lane_id(), w = warp_id();
  __syncthreads();
  const int k0 = blockIdx.x * p.k_per, k1 = min(p.K, k0 + p.k_per), n = max(0, (k1 - k0 + C::KC - 1) / C::KC);
  const T* A = static_cast<const T*>(p.a) + static_cast<long long>(tile.adapter) * p.K * p.R;
  auto load = [&](int c) {
    if (c < n) {
      uint8_t* s = s_ring + c % C::ST * C::STAGE;
      const int k = k0 + c * C::KC;
      for (int i = tid; i < TM * 8; i += kLoraThreads) {
        const int r = i >> 3, ch = i & 7, kk = k + ch * 8;
        const bool in = r < tile.count && kk < k1;
        cp_async16(smem_u32(s + lora_swz<128>(r, ch)), static_cast<const T*>(p.x) + s_row[r] * p.x_stride + (in ? kk : 0), in ? 16 : 0);
      }
      for (int i = tid; i < C::KC * RP / 8; i += kLoraThreads) {
        const int r = i / (RP / 8), ch = i % (RP / 8);
        const bool in = k + r < k1 && ch * 8 < p.R;
        cp_async16(smem_u32(s + C::XB + lora_swz<RP * 2>(r, ch)), A + (in ? static_cast<long long>(k + r) * p.R + ch * 8 : 0), in ? 16 : 0);
      }
    }
    cp_async_commit();
  };
  float acc[RP / 8][4];
#pragma unroll
  for (int i = 0; i < RP / 8; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[i][e] = 0.f;
  for (int c = 0; c < C::ST - 1; ++c) load(c);
  const int mi = lane >> 3, ri = lane & 7, r0 = w * 16;
  for (int c = 0; c < n; ++c) {
    cp_async_wait<C::ST - 2>();
    __syncthreads();
    load(c + C::ST - 1);
    const uint32_t xs = smem_u32(s_ring + c % C::ST * C::STAGE), as = xs + C::XB;
#pragma unroll
    for (int kk = 0; kk < C::KC / 16; ++kk) {
      uint32_t a[4];
      ldsm4(xs + lora_swz<128>(r0 + ri + (mi & 1) * 8, kk * 2 + (mi >> 1)), a);
#pragma unroll
      for (int j = 0; j < RP / 16; ++j) {
        uint32_t b[4];
        ldsm4_t(as + lora_swz<RP * 2>(kk * 16 + ri + (mi & 1) * 8, j * 2 + (mi >> 1)), b);
        mma16816<BF16>(acc[2 * j], a, b[0], b[1]);
        mma16816<BF16>(acc[2 * j + 1], a, b[2], b[3]);
      }
    }
  }
  cp_async_wait<0>();
  __syncthreads();
  const int g = lane >> 2, c2 = (lane & 3) * 2;
  float* s = reinterpret_cast<float*>(s_ring);
#pragma unroll
  for (int j = 0; j < RP / 8; ++j)
#pragma unroll
    for (int e = 0; e < 4; e += 2)
      *reinterpret_cast<float2*>(s + (w * 16 + g + (e >> 1) * 8) * RP + j * 8 + c2) = make_float2(acc[j][e], acc[j][e + 1]);
  lora_meet(s, p.t + static_cast<long long>(tile.at) * RP, tile.count * RP, p.splits);
}

// t of rows g and g + 8 of a warp's 16 as operands of the second product: the 16-bit rounding and the rest, which leave out
// 2^-16 of it in bf16 and 2^-22 in f16 at most.  f16 takes it as multiples `up` of a power of two near the row's largest, so
// that it fits the type.  The rounding is a finite one, so that the rest of an infinite t, or of one that would round to an
// infinity, is what it should be.  at(r, k): t of row r, columns k, k + 1.
template <bool BF16, int RP, typename At>
TKB_DEVFN void lora_split(At&& at, float (&up)[2], uint32_t (&hi)[RP / 16][4], uint32_t (&lo)[RP / 16][4]) {
  const int g = lane_id() >> 2, c2 = (lane_id() & 3) * 2;
  float t[RP / 16][8], top[2] = {0.f, 0.f}, down[2] = {1.f, 1.f};
  up[0] = up[1] = 1.f;
#pragma unroll
  for (int k = 0; k < RP / 16; ++k)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 s = at(g + (i & 1) * 8, k * 16 + (i >> 1) * 8 + c2);
      t[k][2 * i] = s.x;
      t[k][2 * i + 1] = s.y;
      if (!BF16) {
        if (fabsf(s.x) < INFINITY) top[i & 1] = fmaxf(top[i & 1], fabsf(s.x));
        if (fabsf(s.y) < INFINITY) top[i & 1] = fmaxf(top[i & 1], fabsf(s.y));
      }
    }
  if (!BF16) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 1));
      top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 2));
      if (top[i] > 1e-30f && top[i] < 1e30f) {  // else 0, or next to it or to the largest there is
        const int e = (__float_as_int(top[i]) >> 23) - 127;
        up[i] = __int_as_float((e + 127) << 23);
        down[i] = __int_as_float((127 - e) << 23);
      }
    }
  }
#pragma unroll
  for (int k = 0; k < RP / 16; ++k)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      constexpr float MOST = BF16 ? 3.38953139e38f : 65504.f;
      const float a = t[k][2 * i] * down[i & 1], b = t[k][2 * i + 1] * down[i & 1];
      hi[k][i] = pack2<BF16>(fminf(fmaxf(a, -MOST), MOST), fminf(fmaxf(b, -MOST), MOST));
      const float2 h = unpack2<BF16>(hi[k][i]);
      lo[k][i] = pack2<BF16>(a - h.x, b - h.y);
    }
}
// acc = t B for NT8 times 8 columns from piece j0 on of a [RP][64] tile of B.
template <bool BF16, int RP, int NT8>
TKB_DEVFN void lora_columns(uint32_t bs, int j0, const uint32_t (&hi)[RP / 16][4], const uint32_t (&lo)[RP / 16][4],
                            float (&acc)[NT8][4]) {
  const int mi = lane_id() >> 3, ri = lane_id() & 7;
#pragma unroll
  for (int j = 0; j < NT8; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[j][e] = 0.f;
#pragma unroll
  for (int k = 0; k < RP / 16; ++k)
#pragma unroll
    for (int j = 0; j < NT8; j += 2) {
      uint32_t b[4];
      ldsm4_t(bs + lora_swz<128>(k * 16 + ri + (mi & 1) * 8, j0 + j + (mi >> 1)), b);
      mma16816<BF16>(acc[j], hi[k], b[0], b[1]);
      mma16816<BF16>(acc[j + 1], hi[k], b[2], b[3]);
      mma16816<BF16>(acc[j], lo[k], b[0], b[1]);
      mma16816<BF16>(acc[j + 1], lo[k], b[2], b[3]);
    }
}
// acc added to y where it lies in shared memory, rows r0 .., by the threads that hold the products.
template <bool BF16, int NT8>
TKB_DEVFN void lora_onto(uint8_t* ys, int r0, int j0, const float (&up)[2], const float (&acc)[NT8][4]) {
  const int g = lane_id() >> 2, c2 = (lane_id() & 3) * 2;
#pragma unroll
  for (int j = 0; j < NT8; ++j)
#pragma unroll
    for (int e = 0; e < 4; e += 2) {
      uint32_t* at = reinterpret_cast<uint32_t*>(ys + lora_swz<128>(r0 + g + (e >> 1) * 8, j0 + j) + c2 * 2);
      const float2 v = unpack2<BF16>(*at);
      *at = pack2<BF16>(fmaf(acc[j][e], up[e >> 1], v.x), fmaf(acc[j][e + 1], up[e >> 1], v.y));
    }
}

// out = y + t B for one tile of 64 rows and `chunks` times 64 columns, 16 rows a warp.
template <typename T, int RP, int TM>
struct LoraUp {
  static constexpr int NC = 64, ST = 3;
  static constexpr int YB = TM * NC * 2, BB = RP * NC * 2, STAGE = YB + BB, SMEM = ST * STAGE;
};
template <typename T, int RP>
__global__ void __launch_bounds__(kLoraThreads) lora_up_kernel(const __grid_constant__ LoraParams p) {
  constexpr int TM = 64;
  using C = LoraUp<T, RP, TM>;
  constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
  extern __shared__ __align__(128) uint8_t s_ring[];
  __shared__ int s_row[TM];
  grid_wait();
  grid_go();
  const int n_tiles = *p.n_tiles;
  const LoraTile tile = p.tiles[blockIdx.y];
  if (threadIdx.x < TM) s_row[threadIdx.x] = p.row_of[blockIdx.y * TM + threadIdx.x];
  if (static_cast<int>(blockIdx.y) >= n_tiles || (tile.adapter < 0 && p.out == p.y)) return;
  const int tid = threadIdx.x, lane = lane_id(), w = warp_id();
  __syncthreads();
  const int n0 = blockIdx.x * p.chunks * C::NC, n = min(p.chunks, (p.N - n0 + C::NC - 1) / C::NC);
  const T* y = static_cast<const T*>(p.y);
  T* out = static_cast<T*>(p.out);
  if (tile.adapter < 0) {  // no adapter: the rows as they are
    const int pieces = min(n * C::NC, p.N - n0) / 8;
    for (int i = tid; i < tile.count * pieces; i += kLoraThreads) {
      const int r = s_row[i / pieces], col = n0 + i % pieces * 8;
      *reinterpret_cast<uint4*>(out + r * p.out_stride + col) = *reinterpret_cast<const uint4*>(y + r * p.y_stride + col);
    }
    return;
  }
  const T* Bm = static_cast<const T*>(p.b) + static_cast<long long>(tile.adapter) * p.R * p.N;
  auto load = [&](int c) {
    if (c < n) {
      uint8_t* s = s_ring + c % C::ST * C::STAGE;
      const int col = n0 + c * C::NC;
      for (int i = tid; i < TM * 8; i += kLoraThreads) {
        const int r = i >> 3, ch = i & 7, cc = col + ch * 8;
        const bool in = r < tile.count && cc < p.N;
        cp_async16(smem_u32(s + lora_swz<128>(r, ch)), y + s_row[r] * p.y_stride + (in ? cc : 0), in ? 16 : 0);
      }
      for (int i = tid; i < RP * 8; i += kLoraThreads) {
        const int r = i >> 3, ch = i & 7, cc = col + ch * 8;
        const bool in = r < p.R && cc < p.N;
        cp_async16(smem_u32(s + C::YB + lora_swz<128>(r, ch)), Bm + (in ? static_cast<long long>(r) * p.N + cc : 0), in ? 16 : 0);
      }
    }
    cp_async_commit();
  };
  for (int c = 0; c < C::ST - 1; ++c) load(c);
  const int r0 = w * 16;
  const float scale = p.scale ? p.scale[tile.adapter] : 1.f;
  float up[2];
  uint32_t hi[RP / 16][4], lo[RP / 16][4];
  lora_split<BF16, RP>([&](int r, int k) {
    float2 s = make_float2(0.f, 0.f);
    // columns behind the rank are sums of zeros, or of zeros times an infinity
    if (r0 + r < tile.count && k < p.R) s = *reinterpret_cast<const float2*>(p.t + (static_cast<long long>(tile.at) + r0 + r) * RP + k);
    return make_float2(s.x * scale, s.y * scale);
  }, up, hi, lo);
  for (int c = 0; c < n; ++c) {
    cp_async_wait<C::ST - 2>();
    __syncthreads();
    load(c + C::ST - 1);
    uint8_t* ys = s_ring + c % C::ST * C::STAGE;
    float acc[8][4];
    lora_columns<BF16, RP, 8>(smem_u32(ys) + C::YB, 0, hi, lo, acc);
    lora_onto<BF16, 8>(ys, r0, 0, up, acc);
    __syncwarp();
    const int col = n0 + c * C::NC;
#pragma unroll
    for (int i = lane; i < 16 * 8; i += 32) {
      const int r = r0 + (i >> 3), ch = i & 7;
      if (r < tile.count && col + ch * 8 < p.N)
        *reinterpret_cast<uint4*>(out + s_row[r] * p.out_stride + col + ch * 8) = *reinterpret_cast<const uint4*>(ys + lora_swz<128>(r, ch));
    }
  }
  cp_async_wait<0>();
}

// ------------------------------------------------------------ tiles of 16 rows in one kernel
// A cluster per tile: its CTAs take parts of K, sum t through their shared
// memories, and then parts of the columns, whose first loads have been under
// way since the start.  A warp walks over columns on its own, 64 at a time.
template <typename T, int RP>
struct LoraOne {
  static constexpr int ST = RP == 16 ? 3 : 2, STAGE = 16 * 128 + RP * 128;  // per warp: y and B
  static constexpr int DOWN = LoraDown<T, RP, 16>::SMEM, OFF_T = DOWN, OFF_UP = OFF_T + 16 * RP * 4;
  static constexpr int SMEM = OFF_UP + 4 * ST * STAGE;
  static_assert(SMEM <= 232448 - 1024, "shared memory");
};
template <typename T, int RP>
__global__ void __launch_bounds__(kLoraThreads) lora_one_kernel(const __grid_constant__ LoraParams p) {
  using C = LoraOne<T, RP>;
  using Dn = LoraDown<T, RP, 16>;
  constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
  extern __shared__ __align__(128) uint8_t s_ring[];
  __shared__ int s_row[16];
  grid_wait();
  grid_go();
  const int n_tiles = *p.n_tiles;
  const LoraTile tile = p.tiles[blockIdx.y];  // read beside the number: behind it lies what an earlier plan left
  if (threadIdx.x < 16) s_row[threadIdx.x] = p.row_of[blockIdx.y * 16 + threadIdx.x];
  if (static_cast<int>(blockIdx.y) >= n_tiles || (tile.adapter < 0 && p.out == p.y)) return;
  const int tid = threadIdx.x, lane = lane_id(), w = warp_id(), ctas = p.splits, rank = blockIdx.x;
  __syncthreads();
  const T* y = static_cast<const T*>(p.y);
  T* out = static_cast<T*>(p.out);
  const int c0 = rank * p.chunks, c1 = min(c0 + p.chunks, (p.N + 63) / 64);  // chunks of 64 columns
  if (tile.adapter < 0) {  // no adapter: the rows as they are
    const int n0 = c0 * 64, pieces = max(0, min(c1 * 64, p.N) - n0) / 8;
    for (int i = tid; i < tile.count * pieces; i += kLoraThreads) {
      const int r = s_row[i / pieces], col = n0 + i % pieces * 8;
      *reinterpret_cast<uint4*>(out + r * p.out_stride + col) = *reinterpret_cast<const uint4*>(y + r * p.y_stride + col);
    }
    return;
  }
  const T* A = static_cast<const T*>(p.a) + static_cast<long long>(tile.adapter) * p.K * p.R;
  const T* Bm = static_cast<const T*>(p.b) + static_cast<long long>(tile.adapter) * p.R * p.N;
  uint8_t* mine = s_ring + C::OFF_UP + w * C::ST * C::STAGE;
  auto load_up = [&](int i) {  // the warp's i-th chunk
    const int c = c0 + w + 4 * i;
    if (c < c1) {
      uint8_t* s = mine + i % C::ST * C::STAGE;
      for (int e = lane; e < 16 * 8; e += 32) {
        const int r = e >> 3, ch = e & 7, cc = c * 64 + ch * 8;
        const bool in = r < tile.count && cc < p.N;
        cp_async16(smem_u32(s + lora_swz<128>(r, ch)), y + s_row[r] * p.y_stride + (in ? cc : 0), in ? 16 : 0);
      }
      for (int e = lane; e < RP * 8; e += 32) {
        const int r = e >> 3, ch = e & 7, cc = c * 64 + ch * 8;
        const bool in = r < p.R && cc < p.N;
        cp_async16(smem_u32(s + 16 * 128 + lora_swz<128>(r, ch)), Bm + (in ? static_cast<long long>(r) * p.N + cc : 0), in ? 16 : 0);
      }
    }
    cp_async_commit();
  };
  const int k0 = rank * p.k_per, k1 = min(p.K, k0 + p.k_per), n = max(0, (k1 - k0 + Dn::KC - 1) / Dn::KC);
  auto load_down = [&](int c) {
    if (c < n) {
      uint8_t* s = s_ring + c % Dn::ST * Dn::STAGE;
      const int k = k0 + c * Dn::KC, r = tid >> 3, ch = tid & 7, kk = k + ch * 8;
      const bool in = r < tile.count && kk < k1;
      cp_async16(smem_u32(s + lora_swz<128>(r, ch)), static_cast<const T*>(p.x) + s_row[r] * p.x_stride + (in ? kk : 0), in ? 16 : 0);
      for (int i = tid; i < Dn::KC * RP / 8; i += kLoraThreads) {
        const int ar = i / (RP / 8), ac = i % (RP / 8);
        const bool there = k + ar < k1 && ac * 8 < p.R;
        cp_async16(smem_u32(s + Dn::XB + lora_swz<RP * 2>(ar, ac)), A + (there ? static_cast<long long>(k + ar) * p.R + ac * 8 : 0), there ? 16 : 0);
      }
    }
    cp_async_commit();
  };
  // ---- t: this CTA's part of K, a quarter of every chunk a warp
  for (int i = 0; i < C::ST - 1; ++i) load_up(i);
  for (int c = 0; c < Dn::ST - 1; ++c) load_down(c);
  const int mi = lane >> 3, ri = lane & 7, g = lane >> 2, c2 = (lane & 3) * 2;
  {
    float acc[RP / 8][4];
#pragma unroll
    for (int i = 0; i < RP / 8; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i][e] = 0.f;
    for (int c = 0; c < n; ++c) {
      cp_async_wait<Dn::ST - 2>();
      __syncthreads();
      load_down(c + Dn::ST - 1);
      const uint32_t xs = smem_u32(s_ring + c % Dn::ST * Dn::STAGE), as = xs + Dn::XB;
      uint32_t a[4];
      ldsm4(xs + lora_swz<128>(ri + (mi & 1) * 8, w * 2 + (mi >> 1)), a);
#pragma unroll
      for (int j = 0; j < RP / 16; ++j) {
        uint32_t b[4];
        ldsm4_t(as + lora_swz<RP * 2>(w * 16 + ri + (mi & 1) * 8, j * 2 + (mi >> 1)), b);
        mma16816<BF16>(acc[2 * j], a, b[0], b[1]);
        mma16816<BF16>(acc[2 * j + 1], a, b[2], b[3]);
      }
    }
    cp_async_wait<0>();
    __syncthreads();
    float* s = reinterpret_cast<float*>(s_ring);
#pragma unroll
    for (int j = 0; j < RP / 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; e += 2)
        *reinterpret_cast<float2*>(s + (w * 16 + g + (e >> 1) * 8) * RP + j * 8 + c2) = make_float2(acc[j][e], acc[j][e + 1]);
    __syncthreads();
    for (int i = tid; i < 16 * RP; i += kLoraThreads)
      s[64 * RP + i] = (s[i] + s[16 * RP + i]) + (s[32 * RP + i] + s[48 * RP + i]);
    // every CTA sums the cluster's parts for itself, in the order of the ranks
    if (ctas > 1) cluster_sync();
    else __syncthreads();
    const float scale = p.scale ? p.scale[tile.adapter] : 1.f;
    float* st = reinterpret_cast<float*>(s_ring + C::OFF_T);
    const uint32_t here = smem_u32(s + 64 * RP);
    for (int i = tid * 4; i < 16 * RP; i += kLoraThreads * 4) {
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int c = 0; c < ctas; ++c) {
        float4 v;
        if (ctas == 1) v = *reinterpret_cast<const float4*>(s + 64 * RP + i);
        else
          asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                       : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(mapa_shared(here + i * 4, c)) : "memory");
        sum.x += v.x;
        sum.y += v.y;
        sum.z += v.z;
        sum.w += v.w;
      }
      *reinterpret_cast<float4*>(st + i) = make_float4(sum.x * scale, sum.y * scale, sum.z * scale, sum.w * scale);
    }
    __syncthreads();
    if (ctas > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // the others' parts have been read
  }
  // ---- out
  float up[2];
  uint32_t hi[RP / 16][4], lo[RP / 16][4];
  const float* st = reinterpret_cast<const float*>(s_ring + C::OFF_T);
  lora_split<BF16, RP>([&](int r, int k) {
    return k < p.R ? *reinterpret_cast<const float2*>(st + r * RP + k) : make_float2(0.f, 0.f);
  }, up, hi, lo);
  for (int i = 0; c0 + w + 4 * i < c1; ++i) {
    // the chunks asked for at the start are here; from then on the ring's own
    cp_async_wait<C::ST - 2>();
    __syncwarp();
    load_up(i + C::ST - 1);
    uint8_t* ys = mine + i % C::ST * C::STAGE;
    float acc[8][4];
    lora_columns<BF16, RP, 8>(smem_u32(ys) + 16 * 128, 0, hi, lo, acc);
    lora_onto<BF16, 8>(ys, 0, 0, up, acc);
    __syncwarp();
    const int col = (c0 + w + 4 * i) * 64;
#pragma unroll
    for (int e = lane; e < 16 * 8; e += 32) {
      const int r = e >> 3, ch = e & 7;
      if (r < tile.count && col + ch * 8 < p.N)
        *reinterpret_cast<uint4*>(out + s_row[r] * p.out_stride + col + ch * 8) = *reinterpret_cast<const uint4*>(ys + lora_swz<128>(r, ch));
    }
    __syncwarp();  // before the stage is loaded again
  }
  cp_async_wait<0>();
  if (ctas > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // the others have read this CTA's part
}

// ------------------------------------------------------------ fp32: FMA
template <int RP, int TM>
struct LoraDown<float, RP, TM> {
  static constexpr int KC = 32, ST = 3;
  static constexpr int XS = KC + 4;                      // floats from row to row: eight rows in different banks
  static constexpr int XB = TM * XS * 4, AB = KC * RP * 4, STAGE = XB + AB;
  static constexpr int SMEM = ST * STAGE > TM * RP * 4 ? ST * STAGE : TM * RP * 4;
};
template <int RP, int TM>
__global__ void __launch_bounds__(kLoraThreads) lora_down_f32_kernel(const __grid_constant__ LoraParams p) {
  using C = LoraDown<float, RP, TM>;
  constexpr int CG = RP / 4, RG = kLoraThreads / CG < TM ? kLoraThreads / CG : TM, PER = TM / RG;  // threads along R and rows, rows each
  extern __shared__ __align__(128) uint8_t s_ring[];
  __shared__ int s_row[TM];
  grid_wait();
  grid_go();
  const int n_tiles = *p.n_tiles;
  const LoraTile tile = p.tiles[blockIdx.y];  // read beside the number: behind it lies what an earlier plan left
  if (threadIdx.x < TM) s_row[threadIdx.x] = p.row_of[blockIdx.y * TM + threadIdx.x];
  if (static_cast<int>(blockIdx.y) >= n_tiles || tile.adapter < 0) return;
  const int tid = threadIdx.x;
  __syncthreads();
  const int k0 = blockIdx.x * p.k_per, k1 = min(p.K, k0 + p.k_per), n = max(0, (k1 - k0 + C::KC - 1) / C::KC);
  const float* A = static_cast<const float*>(p.a) + static_cast<long long>(tile.adapter) * p.K * p.R;
  auto load = [&](int c) {
    if (c < n) {
      uint8_t* s = s_ring + c % C::ST * C::STAGE;
      const int k = k0 + c * C::KC;
      for (int i = tid; i < TM * 8; i += kLoraThreads) {
        const int r = i >> 3, kk = k + (i & 7) * 4;
        const bool in = r < tile.count && kk < k1;
        cp_async16(smem_u32(s + (r * C::XS + (i & 7) * 4) * 4), static_cast<const float*>(p.x) + s_row[r] * p.x_stride + (in ? kk : 0), in ? 16 : 0);
      }
      for (int i = tid; i < C::KC * RP / 4; i += kLoraThreads) {
        const int r = i / CG, ch = i % CG * 4;
        const bool in = k + r < k1 && ch < p.R;
        cp_async16(smem_u32(s + C::XB + i * 16), A + (in ? static_cast<long long>(k + r) * p.R + ch : 0), in ? 16 : 0);
      }
    }
    cp_async_commit();
  };
  const int cg = tid % CG, rg = tid / CG;
  const bool busy = rg < RG;
  float acc[PER][4];
#pragma unroll
  for (int i = 0; i < PER; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[i][e] = 0.f;
  for (int c = 0; c < C::ST - 1; ++c) load(c);
  for (int c = 0; c < n; ++c) {
    cp_async_wait<C::ST - 2>();
    __syncthreads();
    load(c + C::ST - 1);
    const float* xs = reinterpret_cast<const float*>(s_ring + c % C::ST * C::STAGE);
    const float4* as = reinterpret_cast<const float4*>(s_ring + c % C::ST * C::STAGE + C::XB);
    if (busy)
#pragma unroll 2
      for (int k = 0; k < C::KC; k += 4) {
        float4 a[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) a[e] = as[(k + e) * CG + cg];
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const float4 x = *reinterpret_cast<const float4*>(xs + (i * RG + rg) * C::XS + k);
          const float xv[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            acc[i][0] = fmaf(xv[e], a[e].x, acc[i][0]);
            acc[i][1] = fmaf(xv[e], a[e].y, acc[i][1]);
            acc[i][2] = fmaf(xv[e], a[e].z, acc[i][2]);
            acc[i][3] = fmaf(xv[e], a[e].w, acc[i][3]);
          }
        }
      }
  }
  cp_async_wait<0>();
  __syncthreads();
  float* s = reinterpret_cast<float*>(s_ring);
  if (busy)
#pragma unroll
    for (int i = 0; i < PER; ++i)
      *reinterpret_cast<float4*>(s + (i * RG + rg) * RP + cg * 4) = make_float4(acc[i][0], acc[i][1], acc[i][2], acc[i][3]);
  lora_meet(s, p.t + static_cast<long long>(tile.at) * RP, tile.count * RP, p.splits);
}

template <int RP, int TM>
struct LoraUp<float, RP, TM> {
  static constexpr int NC = 64, TS = RP + 4;
  static constexpr int TB = TM * TS * 4, BB = RP * NC * 4, SMEM = TB + BB;
};
template <int RP, int TM>
__global__ void __launch_bounds__(kLoraThreads) lora_up_f32_kernel(const __grid_constant__ LoraParams p) {
  using C = LoraUp<float, RP, TM>;
  constexpr int PER = TM / 8;  // rows per thread: 16 threads of 4 columns, 8 of rows
  extern __shared__ __align__(128) uint8_t s_ring[];
  __shared__ int s_row[TM];
  grid_wait();
  grid_go();
  const int n_tiles = *p.n_tiles;
  const LoraTile tile = p.tiles[blockIdx.y];
  if (threadIdx.x < TM) s_row[threadIdx.x] = p.row_of[blockIdx.y * TM + threadIdx.x];
  if (static_cast<int>(blockIdx.y) >= n_tiles || (tile.adapter < 0 && p.out == p.y)) return;
  const int tid = threadIdx.x, cg = tid % 16, rg = tid / 16;
  float* ts = reinterpret_cast<float*>(s_ring);
  float* bs = reinterpret_cast<float*>(s_ring + C::TB);
  if (tile.adapter >= 0) {
    const float scale = p.scale ? p.scale[tile.adapter] : 1.f;
    for (int i = tid; i < TM * RP; i += kLoraThreads) {
      const int r = i / RP, k = i % RP;
      ts[r * C::TS + k] = r < tile.count && k < p.R ? p.t[(static_cast<long long>(tile.at) + r) * RP + k] * scale : 0.f;
    }
  }
  const float* y = static_cast<const float*>(p.y);
  float* out = static_cast<float*>(p.out);
  const float* Bm = static_cast<const float*>(p.b) + static_cast<long long>(max(tile.adapter, 0)) * p.R * p.N;
  const int n0 = blockIdx.x * p.chunks * C::NC;
  for (int c = 0; c < p.chunks; ++c) {
    const int base = n0 + c * C::NC, col = base + cg * 4;
    if (base >= p.N) break;
    __syncthreads();
    if (tile.adapter >= 0)
      for (int i = tid; i < RP * 16; i += kLoraThreads) {
        const int r = i / 16, cc = base + i % 16 * 4;
        const bool in = r < p.R && cc < p.N;
        cp_async16(smem_u32(bs + i * 4), Bm + (in ? static_cast<long long>(r) * p.N + cc : 0), in ? 16 : 0);
      }
    cp_async_commit();
    float4 v[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i)
      v[i] = col < p.N && i * 8 + rg < tile.count
                 ? *reinterpret_cast<const float4*>(y + s_row[i * 8 + rg] * p.y_stride + col) : make_float4(0.f, 0.f, 0.f, 0.f);
    cp_async_wait<0>();
    __syncthreads();
    if (tile.adapter >= 0)
#pragma unroll 2
      for (int k = 0; k < RP; k += 4) {
        float4 b[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) b[e] = *reinterpret_cast<const float4*>(bs + (k + e) * C::NC + cg * 4);
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const float4 t = *reinterpret_cast<const float4*>(ts + (i * 8 + rg) * C::TS + k);
          const float tv[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            v[i].x = fmaf(tv[e], b[e].x, v[i].x);
            v[i].y = fmaf(tv[e], b[e].y, v[i].y);
            v[i].z = fmaf(tv[e], b[e].z, v[i].z);
            v[i].w = fmaf(tv[e], b[e].w, v[i].w);
          }
        }
      }
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (col < p.N && i * 8 + rg < tile.count)
        *reinterpret_cast<float4*>(out + s_row[i * 8 + rg] * p.out_stride + col) = v[i];
  }
}

// ------------------------------------------------------------ launches
static int lora_rank(int R) { return R <= 16 ? 16 : R <= 64 ? 64 : 128; }

// CTAs that run at the same time, by their shared memory; twelve an SM at most, by the registers of the kernels that need
// little of it (fp32, 40 a thread).
constexpr int lora_resident(int smem) { return 148 * (232448 / (smem + 1280) < 12 ? 232448 / (smem + 1280) : 12); }

template <typename T, int RP, int TM>
static cudaError_t lora_launch(LoraParams& p, int tiles, cudaStream_t st, unsigned& kernels) {
  const int cols = (p.N + 63) / 64;
  p.splits = 1;
  if constexpr (TM == 16 && sizeof(T) == 2) {
    // Clusters until there are four CTAs an SM, of a chunk of K and of columns each at least.  One, two, four and eight parts,
    // 64 tokens of 16 adapters of 16: K 5632, N 2048 22.6, 13.1, 8.0 and 6.5 us; 1024 x 1024 8.1, 5.8, 4.4, 4.8; 256 x 256 3.4,
    // 4.0, 3.9, 4.6; 256 tokens of 64 adapters, 2048 x 2048 14.8, 9.4, 7.6, 10.9 (four are the rule's).
    while (p.splits < 8 && tiles * 2ll * p.splits <= 148 * 4 && p.K >= 128 * p.splits && cols >= 2 * p.splits) p.splits *= 2;
    p.k_per = ((p.K + p.splits - 1) / p.splits + 63) / 64 * 64;
    p.chunks = (cols + p.splits - 1) / p.splits;
    kernels = 1;
    const cudaError_t e = allow_smem<lora_one_kernel<T, RP>>(LoraOne<T, RP>::SMEM);
    if (e != cudaSuccess) return e;
    return launch_early(lora_one_kernel<T, RP>, dim3(p.splits, tiles), kLoraThreads, LoraOne<T, RP>::SMEM, st, p, p.splits);
  } else {
    // Parts of K: as many CTAs as run at the same time (a few more would be a second wave of their own), each of at
    // least 256 columns, a cluster of eight at most.  12.4 k rows of 2048 and 5632 columns, R = 16: 19 and 45 us in 1.1
    // waves, 15 and 35 in less than one.  Both kernels with one, two, four and eight parts: 1.6 k rows of 33 adapters of 64,
    // 4096 x 4096 86, 49, 39 and 31 us; 800 rows of 8 of 16, K 2048 24.4, 14.2, 9.5, 8.4; K 1024 11.4, 8.5, 7.5, 7.1; K 512
    // 7.6, 7.2, 6.1, 6.1 (four and two are the rule's: short sums leave a microsecond, of which fewer CTAs take less room).
    while (p.splits < 8 && tiles * 2ll * p.splits <= lora_resident(LoraDown<T, RP, TM>::SMEM) && p.K >= 512 * p.splits) p.splits *= 2;
    p.k_per = ((p.K + p.splits - 1) / p.splits + 63) / 64 * 64;
    // Columns of out per CTA: up to 512, while there are three waves of CTAs.  64, 128, 256 and 512 of them: 12 k rows, N
    // 11264 138, 116, 110 and 113 us with x A (the rule: 108); 800 rows, N 2048 8.4, 9.5, 10.5, 14.3 (the rule: 8.4).
    const long long fit = static_cast<long long>(tiles) * cols / (3 * lora_resident(LoraUp<T, RP, TM>::SMEM));
    p.chunks = fit < 1 ? 1 : fit > 8 ? 8 : static_cast<int>(fit);
    const dim3 down(p.splits, tiles), up((cols + p.chunks - 1) / p.chunks, tiles);
    void (*first)(LoraParams);
    void (*second)(LoraParams);
    cudaError_t e;
    if constexpr (sizeof(T) == 4) {
      first = lora_down_f32_kernel<RP, TM>;
      second = lora_up_f32_kernel<RP, TM>;
      e = allow_smem<lora_down_f32_kernel<RP, TM>>(LoraDown<T, RP, TM>::SMEM);
      if (e == cudaSuccess) e = allow_smem<lora_up_f32_kernel<RP, TM>>(LoraUp<T, RP, TM>::SMEM);
    } else {
      first = lora_down_kernel<T, RP>;
      second = lora_up_kernel<T, RP>;
      e = allow_smem<lora_down_kernel<T, RP>>(LoraDown<T, RP, TM>::SMEM);
      if (e == cudaSuccess) e = allow_smem<lora_up_kernel<T, RP>>(LoraUp<T, RP, TM>::SMEM);
    }
    kernels = 2;
    if (e == cudaSuccess) e = launch_early(first, down, kLoraThreads, LoraDown<T, RP, TM>::SMEM, st, p, p.splits);
    if (e == cudaSuccess) e = launch_early(second, up, kLoraThreads, LoraUp<T, RP, TM>::SMEM, st, p);
    return e;
  }
}

template <typename T>
static cudaError_t lora_add_t(LoraParams& p, const LoraPlanAt& plan, cudaStream_t st, unsigned& kernels) {
  const int tiles = plan.tiles, rank = lora_rank(p.R);
#define LAUNCH(RP) return plan.tm == 64 ? lora_launch<T, RP, 64>(p, tiles, st, kernels) : lora_launch<T, RP, 16>(p, tiles, st, kernels)
  if (rank == 16) LAUNCH(16);
  if (rank == 64) LAUNCH(64);
  LAUNCH(128);
#undef LAUNCH
}

}  // namespace tkb
