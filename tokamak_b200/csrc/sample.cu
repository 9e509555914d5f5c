// sample.cu -- one token per row of logits from given uniform numbers:
// temperature, top-k, top-p (nucleus), min-p.
//
// Every token's weight exp(-(max - x)/T) is a whole multiple of 2^-31, so its
// sums are exact 64-bit integers (V <= 2^18 keeps them below 2^49) and the
// token cannot depend on how a sum is cut over threads.  All three
// truncations keep a prefix of the order "falling logit, equal ones by
// index", so a row's kept set is described by a key, the number of tokens of
// exactly that key that stay, and a least weight.
//
// A row belongs to a cluster of C CTAs; each holds its slice in shared memory
// (HBM is read once) and each warp a contiguous chunk of it.  The CTAs agree
// by writing their part into a buffer of their own, one cluster barrier, and
// reading everybody's: every CTA then decides the same from the same numbers.
// The cut of top-k or top-p is found without sorting: a guess brackets it,
// one pass sums what lies above the bracket exactly and lists what lies
// inside, and a radix search over the list gives the cut.  A wrong or too wide
// guess is halved and tried again, so it costs time only.
#include "tkb_common.cuh"

namespace tkb {

struct SampleParams {
  const void* logits;
  long long ld;
  const float* u;
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  int32_t* token;
  float* logprob;
  int32_t* kept;
  int rows, V;
  int per;          // 16-byte vectors per lane: a warp's chunk is per * 32 vectors
  int ctas;         // CTAs per row
};

constexpr int SNT = 256, SW = SNT / 32;
constexpr int SLIST = 256;    // listed elements per warp
constexpr int SBINS = 512;    // bins of the guess, over the distances of non-zero weight
constexpr float SRANGE = 22.25f;  // weights beyond this distance round to zero: 2^31 exp(-22.25) < 1/2

// floor(total * part / 2^32) with part < 2^32
TKB_DEVFN unsigned long long scaled_floor(unsigned long long total, unsigned long long part) {
  return __umul64hi(total, part << 32);
}
TKB_DEVFN unsigned long long scaled_ceil(unsigned long long total, unsigned long long part) {
  return __umul64hi(total, part << 32) + (total * (part << 32) != 0);
}
// A number of [0, 1) as a multiple of 2^-32 (0 for NaN and below, the last one for 1 and above).
TKB_DEVFN unsigned long long fixed32(float x) {
  if (!(x > 0.f)) return 0;
  return x >= 1.f ? 0xFFFFFFFFull : static_cast<unsigned long long>(static_cast<double>(x) * 4294967296.0);
}
// Distance of logit x from its row's maximum in units of the temperature.
TKB_DEVFN float sample_dist(float x, float top, float inv_t) {
  return x == top ? 0.f : __fmul_rn(__fsub_rn(top, x), inv_t);
}
TKB_DEVFN uint32_t sample_weight(float x, float top, float inv_t) {
  return __float2uint_rn(expf(-sample_dist(x, top, inv_t)) * 2147483648.f);
}
// The float of an order_key.
TKB_DEVFN float key_float(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
}

TKB_DEVFN unsigned long long warp_sum_u64(unsigned long long v) {
#pragma unroll
  for (int m = 16; m >= 1; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
  return v;
}

// 8 bytes of shared memory of CTA `rank` of the cluster.
TKB_DEVFN unsigned long long ld_rank_u64(const void* p, int rank) {
  unsigned long long v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(mapa_shared(smem_u32(p), rank)) : "memory");
  return v;
}

template <typename T>
struct Sampler {
  static constexpr int VEC = 16 / sizeof(T);
  const SampleParams& p;
  T* data;                       // the slice
  uint2* list;                   // this warp's (key, index in the row)
  unsigned long long (*xbuf)[256];  // two exchange buffers
  unsigned long long* s_tmp;     // 16 values of the block
  int rank, base, par = 0;       // base: first index of this warp's chunk
  int n_list = 0;                // this warp's listed elements
  bool list_ok = false;          // the elements of the last search's bracket, below list_hi, are listed
  bool summed = false;           // the last pass summed weights
  uint32_t list_hi = 0;
  float top, inv_t;
  unsigned long long above = 0;  // this thread: weight of the elements at list_hi and above
  int n_above = 0;

  TKB_DEVFN Sampler(const SampleParams& q) : p(q) {}

  TKB_DEVFN void vec(int it, float (&x)[VEC]) const {
    ldv<T, VEC>(data + (warp_id() * p.per + it) * 32 * VEC + lane_id() * VEC, x);
  }

  // ---- agreement: fill buf() (after clear() where it is summed into), then agree(), then read()
  TKB_DEVFN unsigned long long* buf() { return xbuf[par]; }
  TKB_DEVFN void clear() {
    xbuf[par][threadIdx.x] = 0;
    __syncthreads();
  }
  TKB_DEVFN void agree() {
    __syncwarp();
    cluster_sync();
  }
  // slot i of CTA r
  TKB_DEVFN unsigned long long read(int i, int r) const { return ld_rank_u64(&xbuf[par][i], r); }
  TKB_DEVFN void next() { par ^= 1; }

  // Two sums over the whole row, known to every thread afterwards.
  TKB_DEVFN void sum2(unsigned long long& a, unsigned long long& b) {
    a = warp_sum_u64(a);
    b = warp_sum_u64(b);
    if (lane_id() == 0) {
      buf()[2 * warp_id()] = a;
      buf()[2 * warp_id() + 1] = b;
    }
    agree();
    a = b = 0;
    // lane l of every warp reads slot pairs l, l + 32, ...
    for (int i = lane_id(); i < p.ctas * SW; i += 32) {
      a += read(2 * (i % SW), i / SW);
      b += read(2 * (i % SW) + 1, i / SW);
    }
    a = warp_sum_u64(a);
    b = warp_sum_u64(b);
    next();
  }

  // One pass over the chunk: what lies at key hi and above is counted (and its
  // weights summed, with `weights`, as are all weights), what lies in
  // [lo, hi) is listed.
  template <bool WEIGHTS>
  TKB_DEVFN void pass(uint32_t lo, uint32_t hi, unsigned long long& in_list, unsigned long long& all) {
    // thresholds as floats; hi one past the largest key means nothing is above
    const float flo = key_float(lo), fhi = key_float(hi);
    n_list = 0;
    n_above = 0;
    summed = WEIGHTS;
    above = in_list = all = 0;
    for (int it = 0; it < p.per; ++it) {
      float x[VEC];
      vec(it, x);
      bool any = false;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const bool is_above = x[e] >= fhi, in = x[e] >= flo && !is_above;
        any |= in;
        n_above += is_above;
        if constexpr (WEIGHTS) {
          const uint32_t w = sample_weight(x[e], top, inv_t);
          all += w;
          if (is_above) above += w;
          if (in) in_list += w;
        } else {
          in_list += in;
        }
      }
      if (__any_sync(0xffffffffu, any)) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const bool in = x[e] >= flo && !(x[e] >= fhi);
          const uint32_t m = __ballot_sync(0xffffffffu, in);
          const int at = n_list + __popc(m & ((1u << lane_id()) - 1));
          if (in && at < SLIST)
            list[at] = make_uint2(order_key(x[e]), base + (it * 32 + lane_id()) * VEC + e);
          n_list += __popc(m);
        }
      }
    }
    __syncwarp();
  }

  // The largest key K of [from, list_hi) such that `acc` and the listed
  // measure of the keys >= K reach `bound` (they do at `from`).  Returns K; acc
  // becomes the measure of the keys above K.
  template <bool WEIGHTS>
  TKB_DEVFN uint32_t radix(uint32_t from, unsigned long long& acc, unsigned long long bound) {
    uint32_t diff = from ^ (list_hi - 1);
    int bits = diff ? 32 - __clz(diff) : 0;
    uint32_t prefix = bits < 32 ? (from >> bits) << bits : 0u;
    while (bits > 0) {
      const int take = bits < 8 ? bits : 8, shift = bits - take;
      clear();
      for (int i = lane_id(); i < n_list; i += 32) {
        const uint32_t key = list[i].x;
        if (key >= from && (bits == 32 || (key >> bits) == (prefix >> bits)))
          atomicAdd(&buf()[(key >> shift) & ((1u << take) - 1)],
                    WEIGHTS ? static_cast<unsigned long long>(sample_weight(key_float(key), top, inv_t)) : 1ull);
      }
      agree();
      // thread t holds digit 255 - t: a prefix sum over threads runs from the largest digit down
      unsigned long long v = 0;
      for (int r = 0; r < p.ctas; ++r) v += read(255 - threadIdx.x, r);
      unsigned long long s = v;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const unsigned long long t = __shfl_up_sync(0xffffffffu, s, d);
        if (lane_id() >= d) s += t;
      }
      if (lane_id() == 31) s_tmp[warp_id()] = s;
      __syncthreads();
      unsigned long long pre = acc;
      for (int i = 0; i < warp_id(); ++i) pre += s_tmp[i];
      s += pre;
      if (s >= bound && s - v < bound) {
        s_tmp[8] = 255 - threadIdx.x;
        s_tmp[9] = s - v;
      }
      __syncthreads();
      prefix |= static_cast<uint32_t>(s_tmp[8]) << shift;
      acc = s_tmp[9];
      __syncthreads();
      next();
      bits = shift;
    }
    return prefix;
  }

  // The cut of a measure (count, or weight): the largest key K of [lo, hi) such
  // that the measure of the keys >= K reaches bound.  False when even lo's does
  // not.  acc: the measure of the keys above the cut.  With of_all the bound
  // comes in as a share, in 2^-32, of the sum of all weights.
  template <bool WEIGHTS>
  TKB_DEVFN bool search(uint32_t lo, uint32_t hi, uint32_t glo, uint32_t ghi, unsigned long long& bound, bool of_all,
                        uint32_t& cut, unsigned long long& acc) {
    while (true) {
      unsigned long long in_list, all;
      pass<WEIGHTS>(glo, ghi, in_list, all);
      unsigned long long a = WEIGHTS ? above : n_above, l = in_list;
      const bool over = n_list > SLIST;
      if (of_all) {
        unsigned long long zero = 0;
        sum2(all, zero);
        bound = scaled_ceil(all, bound);
        if (bound == 0) bound = 1;  // the first token always stays
        of_all = false;
      }
      // the overflow flag rides on the counts' top bits
      unsigned long long flag = over && lane_id() == 0 ? 1ull << 52 : 0ull;
      l += flag;
      sum2(a, l);
      const bool spilled = l >> 52;
      l &= (1ull << 52) - 1;
      if (a >= bound) {
        lo = ghi;
        glo = lo;
        ghi = hi;
      } else if (a + l < bound) {
        if (glo == lo) return false;
        hi = glo;
        glo = lo;
        ghi = hi;
      } else if (!spilled) {
        list_ok = true;
        list_hi = ghi;
        acc = a;
        cut = radix<WEIGHTS>(glo, acc, bound);
        return true;
      } else {
        lo = glo;
        hi = ghi;
        if (hi - lo == 1) {  // one key, more equal logits than the lists hold
          list_ok = false;
          acc = a;
          cut = lo;
          return true;
        }
        glo = lo + (hi - lo) / 2;
      }
    }
  }
};

template <typename T>
__global__ void __launch_bounds__(SNT) sample_kernel(const __grid_constant__ SampleParams p) {
  constexpr int VEC = Sampler<T>::VEC;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ unsigned long long s_x[2][256], s_tmp[16];
  __shared__ uint2 s_list[SW][SLIST];
  Sampler<T> s(p);
  const int row = blockIdx.x / p.ctas, tid = threadIdx.x, lane = lane_id(), w = warp_id(), V = p.V;
  s.rank = blockIdx.x % p.ctas;
  s.data = reinterpret_cast<T*>(smem);
  s.list = s_list[w];
  s.xbuf = s_x;
  s.s_tmp = s_tmp;
  s.base = (s.rank * SW + w) * p.per * 32 * VEC;
  const T* x = static_cast<const T*>(p.logits) + row * p.ld;

  // ---- the slice into shared memory: each lane the vectors it will read
  const bool aligned = (reinterpret_cast<uintptr_t>(x) & 15) == 0;
  for (int it = 0; it < p.per; ++it) {
    const int i = s.base + (it * 32 + lane) * VEC;
    T* dst = s.data + (w * p.per + it) * 32 * VEC + lane * VEC;
    if (aligned && i + VEC <= V) {
      cp_async16(smem_u32(dst), x + i, 16);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        if (i + e < V) dst[e] = x[i + e];
        else Elem<T>::st(dst + e, -INFINITY);
      }
    }
  }
  cp_async_commit();
  cp_async_wait<0>();

  // ---- maximum; NaN becomes -inf for all that follows
  float tmax = -INFINITY;
  for (int it = 0; it < p.per; ++it) {
    float v[VEC];
    s.vec(it, v);
    bool nan = false;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      nan |= v[e] != v[e];
      tmax = fmaxf(tmax, v[e]);
    }
    if (nan) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[e] = v[e] != v[e] ? -INFINITY : v[e];
      stv<T, VEC>(s.data + (w * p.per + it) * 32 * VEC + lane * VEC, v);
    }
  }
  float top = warp_max(tmax);
  if (lane == 0) s.buf()[w] = order_key(top);
  s.agree();
  uint32_t tk = 0;
  for (int i = lane; i < p.ctas * SW; i += 32) tk = max(tk, static_cast<uint32_t>(s.read(i % SW, i / SW)));
  tk = __reduce_max_sync(0xffffffffu, tk);
  s.next();
  top = key_float(tk);
  s.top = top;
  const float temp = p.temperature ? p.temperature[row] : 1.f;
  const bool greedy = !(temp > 0.f);
  s.inv_t = greedy ? 1.f : __frcp_rn(temp);

  if (top == -INFINITY || greedy) {
    // the lowest index of the maximum
    int first = 0x7FFFFFFF;
    if (tmax == top && top > -INFINITY)
      for (int it = p.per - 1; it >= 0; --it) {
        float v[VEC];
        s.vec(it, v);
#pragma unroll
        for (int e = VEC - 1; e >= 0; --e)
          if (v[e] == top) first = s.base + (it * 32 + lane) * VEC + e;
      }
    first = __reduce_min_sync(0xffffffffu, first);
    if (lane == 0) s.buf()[w] = first;
    s.agree();
    int all = 0x7FFFFFFF;
    for (int i = lane; i < p.ctas * SW; i += 32) all = min(all, static_cast<int>(s.read(i % SW, i / SW)));
    all = __reduce_min_sync(0xffffffffu, all);
    if (s.rank == 0 && tid == 0) {
      const bool none = top == -INFINITY;
      p.token[row] = none ? -1 : all;
      if (p.logprob) p.logprob[row] = none ? -INFINITY : 0.f;
      if (p.kept) p.kept[row] = none ? 0 : 1;
    }
    s.agree();  // the others may still read this CTA's buffer
    return;
  }

  const int k = p.top_k && p.top_k[row] > 0 && p.top_k[row] < V ? p.top_k[row] : 0;
  const float tp = p.top_p ? p.top_p[row] : 1.f;
  const bool nucleus = !(tp >= 1.f);
  uint32_t least = 1;
  if (p.min_p && p.min_p[row] > 0.f)
    least = p.min_p[row] >= 1.f ? 0x80000000u
                                : max(1u, static_cast<uint32_t>(ceil(static_cast<double>(p.min_p[row]) * 2147483648.0)));
  // keys of non-zero weight lie in [low, high)
  const uint32_t high = tk + 1;
  const float reach = top - (SRANGE + 1.f) / s.inv_t;
  const uint32_t low = reach == reach ? min(order_key(reach), tk) : order_key(-INFINITY);

  uint32_t cut = 0;  // kept: keys above `cut`, and the first `ties` tokens of exactly that key
  long long ties = 0;
  if (k || nucleus) {
    uint32_t glo = low, ghi = high;
    if (p.per * 32 * VEC > SLIST) {
      // ---- the guess.  Thread maxima enter one by one, a quarter of the other elements stands for the rest.
      uint32_t* hist = reinterpret_cast<uint32_t*>(s.buf());
      s.clear();
      const float to_bin = SBINS / SRANGE;
      const float zmax = sample_dist(tmax, top, s.inv_t);
      const bool by_max = k && k <= p.ctas * SNT / 2;  // enough maxima to bound the k-th largest from below
      if (zmax < SRANGE) atomicAdd(&hist[min(SBINS - 1, static_cast<int>(zmax * to_bin))],
                                   k ? 1u : static_cast<uint32_t>(__expf(-zmax) * 131072.f));
      if (!by_max) {
        const int ns = max(1, p.per / 4);
        const float f = static_cast<float>(p.per) / ns;
        for (int it = 0; it < ns; ++it) {
          float v[VEC];
          s.vec(it, v);
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            const float z = sample_dist(v[e], top, s.inv_t);
            if (v[e] < tmax && z < SRANGE)
              atomicAdd(&hist[min(SBINS - 1, static_cast<int>(z * to_bin))],
                        k ? static_cast<uint32_t>(f + 0.5f) : static_cast<uint32_t>(f * __expf(-z) * 131072.f + 0.5f));
          }
        }
      }
      s.agree();
      // thread t: bins 2t and 2t + 1 of the whole row, and what the bins up to them hold
      unsigned long long h0 = 0, h1 = 0;
      for (int r = 0; r < p.ctas; ++r) {
        const unsigned long long v = s.read(tid, r);
        h0 += v & 0xFFFFFFFFull;
        h1 += v >> 32;
      }
      unsigned long long c = h0 + h1;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const unsigned long long t = __shfl_up_sync(0xffffffffu, c, d);
        if (lane >= d) c += t;
      }
      if (lane == 31) s_tmp[w] = c;
      if (tid == 0) s_tmp[10] = s_tmp[11] = SBINS;
      __syncthreads();
      unsigned long long total = 0;
      for (int i = 0; i < SW; ++i) {
        if (i < w) c += s_tmp[i];
        total += s_tmp[i];
      }
      const unsigned long long c0 = c - h1, b0 = c0 - h0;  // up to and with bin 2t; before it
      double want_lo, want_hi;  // the bracket ends where the estimate passes want_lo, begins where it passes want_hi
      if (by_max) {
        want_lo = k;
        want_hi = -1.0;
      } else if (k) {
        want_lo = 1.2 * k + 8.0 * sqrt(static_cast<double>(k));
        want_hi = -1.0;
      } else {
        // the tail below the cut is sampled well: an error of the sum moves the cut by its share of 1 - p
        const double q = fmax(static_cast<double>(tp), 0.0), room = 0.05 * (1.0 - q) + 1e-4;
        want_lo = (q + room) * total;
        want_hi = (q - room) * total;
      }
      if (c0 >= want_lo && b0 < want_lo) s_tmp[10] = 2 * tid;
      else if (c >= want_lo && c0 < want_lo) s_tmp[10] = 2 * tid + 1;
      if (b0 <= want_hi && c0 > want_hi) s_tmp[11] = 2 * tid;
      else if (c0 <= want_hi && c > want_hi) s_tmp[11] = 2 * tid + 1;
      __syncthreads();
      const int blo = static_cast<int>(s_tmp[10]), bhi = static_cast<int>(s_tmp[11]);
      __syncthreads();
      s.next();
      if (blo < SBINS) {
        const float e = top - (blo + 1) / to_bin / s.inv_t;
        if (e == e) glo = max(low, min(order_key(e), tk));
      }
      if (want_hi > 0 && bhi < SBINS && bhi > 0) {
        const float e = top - bhi / to_bin / s.inv_t;
        if (e == e) ghi = min(high, max(order_key(e), glo + 1));
      }
    }

    auto weight = [&](uint32_t key) -> unsigned long long { return sample_weight(key_float(key), top, s.inv_t); };
    // tokens of key `cut` that stay when the weight above it is acc
    auto ties_of = [&](unsigned long long bound, unsigned long long acc) -> long long {
      const unsigned long long wt = weight(cut);
      return wt ? static_cast<long long>((bound - acc + wt - 1) / wt) : V;
    };
    unsigned long long bound = k, acc = 0;
    bool limited = false;
    if (k) {
      limited = s.template search<false>(low, high, glo, high, bound, false, cut, acc);
      if (limited) ties = k - static_cast<long long>(acc);
    }
    if (nucleus && !limited) {
      // of the whole row (or of fewer than k tokens of any weight)
      bound = fixed32(tp);
      if (s.template search<true>(low, high, k ? low : glo, k ? high : ghi, bound, true, cut, acc)) ties = ties_of(bound, acc);
    } else if (nucleus) {
      // of the first k: their weight above the cut first
      unsigned long long sum = 0, zero = 0;
      const bool listed = s.list_ok && s.list_hi == high;
      if (listed) {
        for (int i = lane; i < s.n_list; i += 32)
          if (s.list[i].x > cut) sum += weight(s.list[i].x);
      } else {
        unsigned long long in_list;
        s.template pass<true>(cut, cut + 1, in_list, zero);
        sum = s.above;
        zero = 0;
        s.list_ok = false;
      }
      s.sum2(sum, zero);
      bound = scaled_ceil(sum + ties * weight(cut), fixed32(tp));
      if (bound == 0) bound = 1;
      if (bound > sum) {
        ties = min(ties, ties_of(bound, sum));
      } else {
        acc = 0;
        if (listed) cut = s.template radix<true>(cut + 1, acc, bound);
        else s.template search<true>(cut + 1, high, cut + 1, high, bound, false, cut, acc);
        ties = ties_of(bound, acc);
      }
    }
  }

  // ---- every warp's kept weight, number kept, and tokens of the cut's own key
  const float fcut = cut ? key_float(cut) : -INFINITY;
  const uint32_t wt = cut ? sample_weight(fcut, top, s.inv_t) : 0u;
  if (wt < least) ties = 0;
  unsigned long long sum = 0;
  unsigned int n_kept = 0, n_tie = 0;
  // the list holds them all, or all that the last pass did not sum already
  const bool listed = s.list_ok && (s.list_hi == high ||
                                    (s.summed && sample_weight(key_float(s.list_hi), top, s.inv_t) >= least));
  if (listed) {
    if (s.list_hi != high) {
      sum = s.above;
      n_kept = s.n_above;
    }
    for (int i = lane; i < s.n_list; i += 32) {
      const uint32_t key = s.list[i].x;
      const uint32_t wi = sample_weight(key_float(key), top, s.inv_t);
      if (key > cut && wi >= least) {
        sum += wi;
        ++n_kept;
      }
      n_tie += key == cut;
    }
  } else {
    for (int it = 0; it < p.per; ++it) {
      float v[VEC];
      s.vec(it, v);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        if (v[e] > fcut) {
          const uint32_t wi = sample_weight(v[e], top, s.inv_t);
          if (wi >= least) {
            sum += wi;
            ++n_kept;
          }
        }
        n_tie += v[e] == fcut;
      }
    }
  }
  sum = warp_sum_u64(sum);
  n_kept = __reduce_add_sync(0xffffffffu, n_kept);
  n_tie = __reduce_add_sync(0xffffffffu, n_tie);
  if (lane == 0) {
    s.buf()[w] = sum;
    s.buf()[SW + w] = (static_cast<unsigned long long>(n_kept) << 32) | n_tie;
  }
  s.agree();
  // lane l: chunks 2l and 2l + 1 of the row's ctas * 8
  unsigned long long cs[2] = {0, 0};
  long long ct[2] = {0, 0}, ck[2] = {0, 0};
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int i = 2 * lane + j;
    if (i < p.ctas * SW) {
      cs[j] = s.read(i % SW, i / SW);
      const unsigned long long v = s.read(SW + i % SW, i / SW);
      ct[j] = static_cast<long long>(v & 0xFFFFFFFFull);
      ck[j] = static_cast<long long>(v >> 32);
    }
  }
  long long tie_pre = ct[0] + ct[1];
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long t = __shfl_up_sync(0xffffffffu, tie_pre, d);
    if (lane >= d) tie_pre += t;
  }
  tie_pre -= ct[0] + ct[1];  // ties before chunk 2l
  const long long stay0 = max(0ll, min(ct[0], ties - tie_pre)), stay1 = max(0ll, min(ct[1], ties - tie_pre - ct[0]));
  cs[0] += stay0 * wt;
  cs[1] += stay1 * wt;
  unsigned long long upto = cs[0] + cs[1];
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const unsigned long long t = __shfl_up_sync(0xffffffffu, upto, d);
    if (lane >= d) upto += t;
  }
  const unsigned long long total = __shfl_sync(0xffffffffu, upto, 31);
  const unsigned long long target = scaled_floor(total, fixed32(p.u[row]));
  const unsigned long long before = upto - cs[0] - cs[1];
  const unsigned kept_all = __reduce_add_sync(0xffffffffu, static_cast<unsigned>(ck[0] + ck[1] + stay0 + stay1));
  const bool in0 = before <= target && target < before + cs[0], in1 = before + cs[0] <= target && target < upto;
  const int owner = __ffs(__ballot_sync(0xffffffffu, in0 || in1)) - 1;
  const int chunk = 2 * owner + __shfl_sync(0xffffffffu, in1 ? 1 : 0, owner);
  unsigned long long run = __shfl_sync(0xffffffffu, in1 ? before + cs[0] : before, owner);
  long long tie_run = __shfl_sync(0xffffffffu, in1 ? tie_pre + ct[0] : tie_pre, owner);

  // ---- the warp whose chunk it is finds the token
  if (chunk == s.rank * SW + w) {
    for (int it = 0; it < p.per; ++it) {
      float v[VEC];
      s.vec(it, v);
      int nt = 0;
#pragma unroll
      for (int e = 0; e < VEC; ++e) nt += v[e] == fcut;
      int pre = nt;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, pre, d);
        if (lane >= d) pre += t;
      }
      const int all_ties = __shfl_sync(0xffffffffu, pre, 31);
      long long rank = tie_run + pre - nt;
      uint32_t we[VEC];
      unsigned long long mine = 0;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const bool tie = v[e] == fcut;
        const uint32_t wi = sample_weight(v[e], top, s.inv_t);
        we[e] = wi >= least && (v[e] > fcut || (tie && rank < ties)) ? wi : 0u;
        rank += tie;
        mine += we[e];
      }
      unsigned long long end = mine;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const unsigned long long t = __shfl_up_sync(0xffffffffu, end, d);
        if (lane >= d) end += t;
      }
      end += run;
      if (end > target && end - mine <= target) {
        unsigned long long at = end - mine;
        int e = 0;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          at += we[i];
          if (at <= target) e = i + 1;
        }
        const int token = s.base + (it * 32 + lane) * VEC + e;
        float xe = v[0];
#pragma unroll
        for (int i = 1; i < VEC; ++i)
          if (i == e) xe = v[i];
        p.token[row] = token;
        if (p.kept) p.kept[row] = static_cast<int32_t>(kept_all);
        if (p.logprob)
          p.logprob[row] = -sample_dist(xe, top, s.inv_t) - logf(static_cast<float>(total) * 4.656612873077393e-10f);
      }
      run = __shfl_sync(0xffffffffu, end, 31);
      tie_run += all_ties;
      if (run > target) break;
    }
  }
  s.agree();  // the others may still read this CTA's buffer
}

constexpr int kSampleMaxV = 1 << 18;

// CTAs per row and vectors per lane.  Slices of 32 KB leave room for four CTAs
// per SM, whose barriers and passes overlap; few rows are cut finer, down to
// one vector per lane, until there are two CTAs per SM.  Eight CTAs is the
// portable cluster size.
static void sample_shape(int rows, int V, int esize, int& ctas, int& per) {
  const int vec = 16 / esize, chunk = SW * 32 * vec;  // elements per CTA and vector
  ctas = 1;
  while (ctas < 8 && (static_cast<long long>(V) * esize > static_cast<long long>(ctas) * 32768 ||
                      (static_cast<long long>(rows) * ctas * 2 <= 296 && V > ctas * chunk)))
    ctas *= 2;
  per = (V + ctas * chunk - 1) / (ctas * chunk);
}

template <typename T>
static cudaError_t sample_t(SampleParams p, cudaStream_t st) {
  sample_shape(p.rows, p.V, sizeof(T), p.ctas, p.per);
  const size_t smem = static_cast<size_t>(p.per) * SNT * 16;
  auto k = sample_kernel<T>;
  cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.rows) * p.ctas);
  cfg.blockDim = dim3(SNT);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = p.ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, k, p);
}

}  // namespace tkb
