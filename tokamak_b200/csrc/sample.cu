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
// When there are rows enough to fill the GPU with one CTA each, a row has one
// CTA of 512 threads (STREAM) that reads it again from L2 in every pass
// instead: no cluster to wait for, and a row's fixed work is done by 16 warps
// instead of 64.
// The cut of top-k or top-p is found without sorting: a guess brackets it,
// one pass sums what lies above the bracket exactly and lists what lies
// inside, and a radix search over the list gives the cut (or, when the list
// holds the row's largest and no more than 256 of them, each is compared with
// all the others).  A guess that missed costs another pass, nothing else.
//
// Measured (us): one row of 32000 bf16, top-k and top-p: 10; 64 rows of 32000
// fp32: 13; 512 rows of 131072 bf16, top-p 0.9 (134 MB): 194.  The last has 48
// instructions per logit, 20 of them in the exponential that the sum of all
// weights needs, which issue in 0.61 of the cycles (87 us of them at full
// rate); most of the rest waits for the vector that a pass has just asked for,
// and for SMs that have four rows where others have three.  Bitwise searches
// re-reading the row took 452, 448 and 5482.
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

constexpr int SCTAS = 8;      // CTAs per row at most: the portable cluster size
constexpr int SSMALL = 256;   // listed elements of a row that are ranked directly, one per thread
constexpr int SBINS = 512;    // bins of the guess, over the distances of non-zero weight
constexpr int kSampleMaxV = 1 << 18;
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
// order_key without the bits that no value of the type has: 16-bit logits need
// half the steps of a search over keys.
template <typename T>
struct SampleKey {
  static constexpr int DROP = sizeof(T) == 4 ? 0 : std::is_same<T, __half>::value ? 13 : 16;
  static TKB_DEVFN uint32_t of(float x) { return order_key(x) >> DROP; }
  static TKB_DEVFN float value(uint32_t key) {
    const uint32_t k = key << DROP;
    return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~(k | ((1u << DROP) - 1)));
  }
};

TKB_DEVFN unsigned long long warp_sum_u64(unsigned long long v) {
#pragma unroll
  for (int m = 16; m >= 1; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
  return v;
}

// 8 bytes of shared memory of CTA `rank` of the cluster.
TKB_DEVFN unsigned long long ld_rank_u64(const void* p, int rank) {
  unsigned long long v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(mapa_shared(smem_u32(p), rank)));
  return v;
}

template <typename T, bool STREAM>
struct Sampler {
  static constexpr int VEC = 16 / sizeof(T);
  static constexpr int NTH = STREAM ? 512 : 256, SW = NTH / 32;
  static constexpr int CTAS = STREAM ? 1 : SCTAS;   // at most
  static constexpr int SLIST = STREAM ? 768 : 256;  // listed elements per warp
  using Key = SampleKey<T>;
  const SampleParams& p;
  T* data;                       // the slice (STREAM: the row)
  bool aligned = true, dirty = false;  // STREAM: 16-byte loads are possible; the row has NaN
  uint2* list;                   // this warp's (key, index in the row)
  unsigned long long (*xbuf)[256];  // two exchange buffers
  unsigned long long* s_tmp;     // 16 values of the block
  int rank, base, par = 0;       // base: first index of this warp's chunk
  int n_list = 0;                // this warp's listed elements
  bool list_ok = false;          // the elements of the last search's bracket, below list_hi, are listed
  bool summed = false;           // the last pass summed weights
  uint32_t list_hi = 0;
  float top, inv_t;
  bool plain = true;             // both finite, 1/T not 0
  unsigned long long above = 0;  // this thread: weight of the elements at list_hi and above
  int n_above = 0;

  TKB_DEVFN Sampler(const SampleParams& q) : p(q) {}

  TKB_DEVFN void vec(int it, float (&x)[VEC]) const {
    at(warp_id(), it, x);
  }
  // this lane's elements of vector `it` of warp w
  TKB_DEVFN void at(int w, int it, float (&x)[VEC]) const {
    const int i = ((w * p.per + it) * 32 + lane_id()) * VEC;
    if constexpr (!STREAM) {
      ldv<T, VEC>(data + i, x);
    } else {
      if (aligned && i + VEC <= p.V) {
        const uint4 q = ld_stream_v4(reinterpret_cast<const uint4*>(data + i));
        ldv<T, VEC>(reinterpret_cast<const T*>(&q), x);
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) x[e] = i + e < p.V ? Elem<T>::ld(data + i + e) : -INFINITY;
      }
      if (dirty)
#pragma unroll
        for (int e = 0; e < VEC; ++e) x[e] = x[e] != x[e] ? -INFINITY : x[e];
    }
  }

  // ---- agreement: fill buf() (after clear() where it is summed into), then agree(), then read()
  TKB_DEVFN unsigned long long* buf() { return xbuf[par]; }
  TKB_DEVFN void clear() {
    if (threadIdx.x < 256) xbuf[par][threadIdx.x] = 0;
    __syncthreads();
  }
  TKB_DEVFN void agree() {
    __syncwarp();
    if constexpr (STREAM) __syncthreads();
    else cluster_sync();
  }
  // slot i of CTA r, and of all CTAs (their loads in flight together)
  TKB_DEVFN unsigned long long read(int i, int r) const {
    if constexpr (STREAM) return xbuf[par][i];
    else return ld_rank_u64(&xbuf[par][i], r);
  }
  TKB_DEVFN void read_all(int i, unsigned long long (&v)[CTAS]) const {
#pragma unroll
    for (int r = 0; r < CTAS; ++r) v[r] = r < p.ctas && i >= 0 && i < 256 ? read(i, r) : 0;
  }
  TKB_DEVFN void next() { par ^= 1; }

  // N sums over the whole row, known to every thread afterwards.
  template <int N>
  TKB_DEVFN void sums(unsigned long long (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = warp_sum_u64(v[i]);
      if (lane_id() == 0) buf()[N * warp_id() + i] = v[i];
    }
    agree();
    const int j0 = lane_id(), j1 = lane_id() + 32;  // the row's warps, at most 64
    unsigned long long a[N], b[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      a[i] = j0 < p.ctas * SW ? read(N * (j0 % SW) + i, j0 / SW) : 0;
      b[i] = j1 < p.ctas * SW ? read(N * (j1 % SW) + i, j1 / SW) : 0;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = a[i] + b[i];
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = warp_sum_u64(v[i]);
    next();
  }

  // One pass over the chunk: what lies at key hi and above is counted (and its
  // weights summed, with WEIGHTS, as are all weights), what lies in [lo, hi) is
  // listed.  `in_list`: the measure of the listed elements, of no meaning when
  // the list spilled.  PLAIN: maximum and 1/T are finite, so that no distance
  // needs a special case.
  //
  // A weight is rint(e 2^31) for e in [0, 1], without a conversion: t = e + 1
  // rounds e to multiples of 2^-23, which are then the low bits of t; the rest,
  // exact, becomes the low bits of rest + 1.5 2^-8 as a multiple of 2^-31.
  // (The conversion unit also computes ex2; it would be the bound.)
  //
  // A lane's upper parts add up to 2^23 for each weight near 2^31, in 32 bits:
  // 512 of them, all that a lane can have (one CTA per row, V near 2^18), make
  // 2^32, which is 0 again.  No other sum of 512 is, but that of weights below
  // 2^7 alone, so one of the lane's elements tells the two apart.  (Adding to 64
  // bits every 256 elements inside the loop cost 4 % of the pass.)
  template <bool WEIGHTS, bool PLAIN>
  TKB_DEVFN void pass_t(uint32_t lo, uint32_t hi, unsigned long long& in_list, unsigned long long& all) {
    // thresholds as floats; hi one past the largest key means nothing is above
    const float flo = Key::value(lo), fhi = Key::value(hi);
    constexpr uint32_t ONE = 0x3F800000u, LOW = 0x3BC00000u;  // 1, 1.5 * 2^-8
    uint32_t hi_all = 0, lo_all = 0, hi_above = 0, lo_above = 0, n = 0, n_in = 0;
    // the vectors with listed elements, as (vector << 8 | mask), from the end of the list's memory downwards
    uint32_t* marks = reinterpret_cast<uint32_t*>(list + SLIST) - 1;
    int n_marks = 0;
    summed = WEIGHTS;
    const uint64_t top2 = f2(top, top), inv2 = f2(inv_t, inv_t), one2 = f2(1.f, 1.f), low2 = f2(0.005859375f, 0.005859375f);
    for (int it = 0; it < p.per; ++it) {
      float x[VEC];
      vec(it, x);
      uint32_t in = 0;  // this lane's elements of the bracket
#pragma unroll
      for (int e = 0; e < VEC; e += 2) {
        const bool above0 = x[e] >= fhi, above1 = x[e + 1] >= fhi;
        if (x[e] >= flo && !above0) in |= 1u << e;
        if (x[e + 1] >= flo && !above1) in |= 2u << e;
        n += above0;
        n += above1;
        if constexpr (WEIGHTS) {
          float z0, z1;
          if constexpr (PLAIN) {
            f2_split(mul_f2(sub_f2(top2, f2(x[e], x[e + 1])), inv2), z0, z1);
          } else {
            z0 = sample_dist(x[e], top, inv_t);
            z1 = sample_dist(x[e + 1], top, inv_t);
          }
          float e0 = expf(-z0), e1 = expf(-z1);
          if constexpr (!PLAIN) {  // -inf logits at an infinite temperature
            e0 = e0 == e0 ? e0 : 0.f;
            e1 = e1 == e1 ? e1 : 0.f;
          }
          const uint64_t ex = f2(e0, e1), t = add_f2(ex, one2);
          const uint64_t l = add_f2(sub_f2(ex, sub_f2(t, one2)), low2);
          float t0, t1, l0, l1;
          f2_split(t, t0, t1);
          f2_split(l, l0, l1);
          hi_all += __float_as_uint(t0) + __float_as_uint(t1);
          lo_all += __float_as_uint(l0) + __float_as_uint(l1);
          if (above0) {
            hi_above += __float_as_uint(t0);
            lo_above += __float_as_uint(l0);
          }
          if (above1) {
            hi_above += __float_as_uint(t1);
            lo_above += __float_as_uint(l1);
          }
        }
      }
      const unsigned m = __ballot_sync(0xffffffffu, in);
      if (m) {
        const int at = n_marks + __popc(m & ((1u << lane_id()) - 1));
        if (in && at < 2 * SLIST) *(marks - at) = static_cast<uint32_t>(it * 32 + lane_id()) << 8 | in;
        n_marks += __popc(m);
        n_in += __popc(in);
      }
    }
    n_list = __reduce_add_sync(0xffffffffu, n_in);
    __syncwarp();
    // From marks to elements, in place, the lowest mark (the last one) first:
    // every mark still unread stands for one element at least, so what is
    // written (8 bytes an element, from the front) ends before the unread marks
    // (4 bytes each, up to the end) begin.
    if (n_list <= SLIST) {
      int done = 0;
      for (int i = 0; i < n_marks; i += 32) {
        uint32_t mark = i + lane_id() < n_marks ? *(marks - (n_marks - 1 - i - lane_id())) : 0u;
        const int mine = __popc(mark & 0xFFu);
        int end = mine;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const int o = __shfl_up_sync(0xffffffffu, end, d);
          if (lane_id() >= d) end += o;
        }
        const int first = static_cast<int>(mark >> 8) * VEC;
        int at = done + end - mine;
        __syncwarp();
        for (mark &= 0xFFu; mark && at < SLIST; mark &= mark - 1, ++at) {
          const int j = base + first + __ffs(mark) - 1;
          const float v = STREAM && j >= p.V ? -INFINITY : Elem<T>::ld(data + (STREAM ? j : j - rank * SW * p.per * 32 * VEC));
          list[at] = make_uint2(Key::of(v), j);
        }
        done += __shfl_sync(0xffffffffu, end, 31);
        __syncwarp();
      }
    }
    n_above = n;
    auto joined = [](uint32_t h, uint32_t l, uint32_t count) {
      return (static_cast<unsigned long long>(h - count * ONE) << 8) +
             static_cast<unsigned long long>(static_cast<long long>(static_cast<int>(l - count * LOW)));
    };
    all = WEIGHTS ? joined(hi_all, lo_all, p.per * VEC) : 0;
    above = WEIGHTS ? joined(hi_above, lo_above, n) : 0;
    if constexpr (WEIGHTS && STREAM) {
      constexpr uint32_t MOST = kSampleMaxV / NTH;  // elements per lane
      static_assert((1ull << 23) * MOST <= 1ull << 32, "a lane's sum wraps at its end at most");
      if (p.per * VEC == MOST) {
        float x[VEC];
        vec(0, x);
        if (hi_all == MOST * ONE && sample_weight(x[0], top, inv_t) >> 30) all += 1ull << 40;
        if (n == MOST) above = all;
      }
    }
    __syncwarp();
    in_list = 0;
    for (int i = lane_id(); i < min(n_list, SLIST); i += 32) in_list += WEIGHTS ? weight_of(list[i].x) : 1u;
  }
  template <bool WEIGHTS>
  TKB_DEVFN void pass(uint32_t lo, uint32_t hi, unsigned long long& in_list, unsigned long long& all) {
    if (!WEIGHTS || plain) pass_t<WEIGHTS, true>(lo, hi, in_list, all);
    else pass_t<WEIGHTS, false>(lo, hi, in_list, all);
  }
  TKB_DEVFN uint32_t weight_of(uint32_t key) const { return sample_weight(Key::value(key), top, inv_t); }

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
        if (key >= from && (bits == 32 || (key >> bits) == (prefix >> bits))) {
          // the sum as two 32-bit ones, of the weights' lower and upper halves (at most SW * SLIST terms each): a 64-bit
          // add to shared memory is a loop
          uint32_t* slot = reinterpret_cast<uint32_t*>(&buf()[(key >> shift) & ((1u << take) - 1)]);
          const uint32_t wt = WEIGHTS ? weight_of(key) : 1u;
          atomicAdd(slot, wt & 0xFFFFu);
          if (WEIGHTS) atomicAdd(slot + 1, wt >> 16);
        }
      }
      agree();
      // thread t holds digit 255 - t: a prefix sum over threads runs from the largest digit down
      unsigned long long part[CTAS], v = 0;
      read_all(255 - static_cast<int>(threadIdx.x), part);
#pragma unroll
      for (int r = 0; r < CTAS; ++r) v += (part[r] & 0xFFFFFFFFull) + ((part[r] >> 32) << 16);
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
        s_tmp[2 * SW] = 255 - threadIdx.x;
        s_tmp[2 * SW + 1] = s - v;
      }
      __syncthreads();
      prefix |= static_cast<uint32_t>(s_tmp[2 * SW]) << shift;
      acc = s_tmp[2 * SW + 1];
      __syncthreads();
      next();
      bits = shift;
    }
    return prefix;
  }

  // The cut of a measure (count, or weight): the largest key K of [lo, hi) such
  // that the measure of the keys >= K reaches bound; acc becomes the measure of
  // the keys above it.  With of_all the bound comes in as a share, in 2^-32, of
  // the sum of all weights.  NONE: even lo's measure does not reach it.  FEW:
  // no cut was looked for, since the lists hold all keys from one at or below
  // the cut up to hi, and they are no more than SSMALL.
  enum { NONE, CUT, FEW };
  template <bool WEIGHTS>
  TKB_DEVFN int search(uint32_t lo, uint32_t hi, uint32_t glo, uint32_t ghi, unsigned long long& bound, bool of_all,
                       uint32_t& cut, unsigned long long& acc) {
    const uint32_t end = hi;
    while (true) {
      unsigned long long in_list, all;
      pass<WEIGHTS>(glo, ghi, in_list, all);
      unsigned long long v[4] = {WEIGHTS ? above : n_above, in_list, 0, all};
      if (lane_id() == 0) v[2] = n_list + (n_list > SLIST ? 1ull << 32 : 0ull);
      sums(v);
      const unsigned long long a = v[0], listed = v[2] & 0xFFFFFFFFull;
      const bool spilled = v[2] >> 32, single = ghi - glo == 1;
      if (of_all) bound = max(1ull, scaled_ceil(v[3], bound));  // the first token always stays
      of_all = false;
      // what the list measures, as far as it is known when it spilled
      unsigned long long l = v[1];
      if (spilled) l = !WEIGHTS ? listed : listed * weight_of(glo);
      // a guess that missed is followed by its neighbour, as wide as what is missing (or too much) would be at the
      // listed measure per key, and half as much again
      const double miss = (a >= bound ? a - bound : bound - a - l) / (static_cast<double>(l) + 1.0);
      const uint32_t wide = 1 + static_cast<uint32_t>(fmin((ghi - glo) * (1.5 * miss + 0.25), 1e9));
      if (a >= bound) {
        lo = ghi;
        glo = lo;
        ghi = hi - lo > wide ? lo + wide : hi;
      } else if (spilled && WEIGHTS && !single) {
        // of the bracket, the upper part that the lists should hold
        const double part = fmin(0.5, 0.4 * p.ctas * SW * SLIST / static_cast<double>(listed));
        hi = ghi;
        glo = ghi - max(1u, static_cast<uint32_t>((ghi - glo) * part));
      } else if (a + l < bound) {
        if (glo == lo) return NONE;
        hi = glo;
        glo = hi - lo > wide ? hi - wide : lo;
        ghi = hi;
      } else if (!spilled) {
        list_ok = true;
        list_hi = ghi;
        if (ghi == end && listed <= SSMALL) return FEW;
        acc = a;
        cut = radix<WEIGHTS>(glo, acc, bound);
        return CUT;
      } else if (single) {  // one key, more equal logits than the lists hold
        list_ok = false;
        acc = a;
        cut = glo;
        return CUT;
      } else {
        lo = glo;
        hi = ghi;
        glo = lo + (hi - lo) / 2;
      }
    }
  }

  // The whole row decided from no more than SSMALL listed elements, the row's
  // largest: they are brought to CTA 0, each of whose threads compares one of
  // them with all the others.
  // bound: what top-p leaves (0: its share of the first k's weight).
  TKB_DEVFN void few(int row, int k, bool nucleus, float tp, unsigned long long bound, uint32_t least, uint4* s_few) {
    const int lane = lane_id(), tid = threadIdx.x;
    if (lane == 0) buf()[warp_id()] = n_list;
    agree();
    int c[2] = {0, 0};
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int i = 2 * lane + j;
      if (i < p.ctas * SW) c[j] = static_cast<int>(read(i % SW, i / SW));
    }
    int end = c[0] + c[1];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int t = __shfl_up_sync(0xffffffffu, end, d);
      if (lane >= d) end += t;
    }
    const int n = __shfl_sync(0xffffffffu, end, 31), mine = rank * SW + warp_id();
    const int at = __shfl_sync(0xffffffffu, end - c[0] - c[1], mine / 2) +
                   (mine & 1 ? __shfl_sync(0xffffffffu, c[0], mine / 2) : 0);
    // (key, index, weight, kept weight) of each
    const uint32_t dst = mapa_shared(smem_u32(s_few), 0);
    for (int i = lane; i < n_list; i += 32)
      if (STREAM) s_few[at + i] = make_uint4(list[i].x, list[i].y, 0u, 0u);
      else asm volatile("st.shared::cluster.v2.u32 [%0], {%1, %2};" ::"r"(dst + 16 * (at + i)), "r"(list[i].x), "r"(list[i].y)
                        : "memory");
    next();
    agree();
    if (rank != 0) return;
    const bool mine_in = warp_id() * 32 < n;  // warps past the list only take part in the sums
    const uint4 e = tid < n ? s_few[tid] : make_uint4(0u, 0u, 0u, 0u);
    const uint32_t wt = tid < n ? weight_of(e.x) : 0u;
    if (tid < n) s_few[tid].z = wt;
    __syncthreads();
    // tokens before this one in the order of the truncations, and their weight
    int rank_of = 0;
    unsigned long long before = 0;
    if (mine_in) {
#pragma unroll 8
      for (int j = 0; j < n; ++j) {
        const uint4 o = s_few[j];
        if (o.x > e.x || (o.x == e.x && o.y < e.y)) {
          ++rank_of;
          before += o.z;
        }
      }
    }
    bool keep = tid < n && (k == 0 || rank_of < k);
    if (nucleus) {
      const unsigned long long total = block_sum(keep ? wt : 0ull);
      if (bound == 0) bound = max(1ull, scaled_ceil(total, fixed32(tp)));
      keep = keep && before < bound;
    }
    keep = keep && wt >= least;
    if (tid < n) s_few[tid].w = keep ? wt : 0u;
    // weights in the lower 52 bits, the number kept above them (its barriers publish s_few)
    const unsigned long long sum = block_sum(keep ? wt | 1ull << 52 : 0ull), total = sum & ((1ull << 52) - 1);
    const unsigned long long target = scaled_floor(total, fixed32(p.u[row]));
    if (!mine_in) return;
    unsigned long long run = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) {
      const uint4 o = s_few[j];
      if (o.y < e.y) run += o.w;
    }
    if (keep && run <= target && target < run + wt) finish(row, e.y, Key::value(e.x), total, static_cast<int>(sum >> 52));
  }
  TKB_DEVFN unsigned long long block_sum(unsigned long long v) {
    v = warp_sum_u64(v);
    __syncthreads();
    if (lane_id() == 0) s_tmp[warp_id()] = v;
    __syncthreads();
    unsigned long long s = 0;
#pragma unroll
    for (int i = 0; i < SW; ++i) s += s_tmp[i];
    return s;
  }
  TKB_DEVFN void finish(int row, int token, float x, unsigned long long total, int kept) {
    p.token[row] = token;
    if (p.kept) p.kept[row] = kept;
    if (p.logprob)
      p.logprob[row] = -sample_dist(x, top, inv_t) - logf(static_cast<float>(total) * 4.656612873077393e-10f);
  }
};

// Larger of two packed pairs, NaN if either is.
template <typename T>
TKB_DEVFN uint32_t max_nan2(uint32_t a, uint32_t b) {
  uint32_t r;
  if constexpr (std::is_same<T, __half>::value) asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

template <typename T, bool STREAM>
__global__ void __launch_bounds__(Sampler<T, STREAM>::NTH, 1024 / Sampler<T, STREAM>::NTH) sample_kernel(const __grid_constant__ SampleParams p) {
  using S = Sampler<T, STREAM>;
  constexpr int VEC = S::VEC, SW = S::SW, SLIST = S::SLIST, CTAS = S::CTAS;
  using Key = SampleKey<T>;
  extern __shared__ __align__(16) uint8_t smem[];  // the lists, then the slice (STREAM: what few() gathers)
  __shared__ unsigned long long s_x[2][256], s_tmp[2 * SW + 8];
  grid_wait();
  S s(p);
  const int row = blockIdx.x / p.ctas, tid = threadIdx.x, lane = lane_id(), w = warp_id(), V = p.V;
  s.rank = blockIdx.x % p.ctas;
  s.list = reinterpret_cast<uint2*>(smem) + w * SLIST;
  s.xbuf = s_x;
  s.s_tmp = s_tmp;
  s.base = (s.rank * SW + w) * p.per * 32 * VEC;
  const T* x = static_cast<const T*>(p.logits) + row * p.ld;
  s.aligned = (reinterpret_cast<uintptr_t>(x) & 15) == 0;
  if constexpr (STREAM) {
    s.data = const_cast<T*>(x);
  } else {
    // ---- the slice into shared memory: each lane the vectors it will read
    s.data = reinterpret_cast<T*>(smem + SW * SLIST * sizeof(uint2));
    for (int it = 0; it < p.per; ++it) {
      const int i = s.base + (it * 32 + lane) * VEC;
      T* dst = s.data + (w * p.per + it) * 32 * VEC + lane * VEC;
      if (s.aligned && i + VEC <= V) {
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
  }

  // ---- maximum; NaN becomes -inf for all that follows
  float tmax = -INFINITY;
  {
    uint32_t m = sizeof(T) == 4 ? 0u : std::is_same<T, __half>::value ? 0xFC00FC00u : 0xFF80FF80u;  // -inf
#pragma unroll(STREAM ? 8 : 1)
    for (int it = 0; it < p.per; ++it) {
      const int i = ((w * p.per + it) * 32 + lane) * VEC;
      if (sizeof(T) == 2 && (!STREAM || (s.aligned && i + VEC <= V))) {
        const uint4* at = reinterpret_cast<const uint4*>(s.data + i);
        const uint4 q = STREAM ? ld_stream_v4(at) : *at;
        m = max_nan2<T>(max_nan2<T>(m, max_nan2<T>(q.x, q.y)), max_nan2<T>(q.z, q.w));
      } else {
        float v[VEC];
        s.vec(it, v);
#pragma unroll
        for (int e = 0; e < VEC; ++e) asm("max.NaN.f32 %0, %1, %2;" : "=f"(tmax) : "f"(tmax), "f"(v[e]));
      }
    }
    if constexpr (sizeof(T) == 2) {
      const float2 f = unpack2<std::is_same<T, __nv_bfloat16>::value>(m);
      asm("max.NaN.f32 %0, %1, %2;" : "=f"(tmax) : "f"(tmax), "f"(f.x));
      asm("max.NaN.f32 %0, %1, %2;" : "=f"(tmax) : "f"(tmax), "f"(f.y));
    }
  }
  if constexpr (STREAM) s.dirty = __syncthreads_or(tmax != tmax);
  if (tmax != tmax) {
    tmax = -INFINITY;
    for (int it = 0; it < p.per; ++it) {
      float v[VEC];
      s.vec(it, v);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        v[e] = v[e] != v[e] ? -INFINITY : v[e];
        tmax = fmaxf(tmax, v[e]);
      }
      if constexpr (!STREAM) stv<T, VEC>(s.data + (w * p.per + it) * 32 * VEC + lane * VEC, v);
    }
  }
  float top = warp_max(tmax);
  if (lane == 0) s.buf()[w] = Key::of(top);
  s.agree();
  uint32_t tk = 0;
  for (int i = lane; i < p.ctas * SW; i += 32) tk = max(tk, static_cast<uint32_t>(s.read(i % SW, i / SW)));
  tk = __reduce_max_sync(0xffffffffu, tk);
  s.next();
  top = Key::value(tk);
  s.top = top;
  const float temp = p.temperature ? p.temperature[row] : 1.f;
  const bool greedy = !(temp > 0.f);
  s.inv_t = greedy ? 1.f : __frcp_rn(temp);
  s.plain = top < INFINITY && s.inv_t < INFINITY && s.inv_t > 0.f;

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
  const uint32_t low = reach == reach ? min(Key::of(reach), tk) : Key::of(-INFINITY);

  uint32_t cut = 0;  // kept: keys above `cut`, and the first `ties` tokens of exactly that key
  long long ties = 0;
  if (k || nucleus) {
    uint32_t glo = low, ghi = high;
    if (p.per * 32 * VEC > SLIST) {
      // ---- the guess.  Thread maxima enter one by one, an eighth of the other elements stands for the rest.
      uint32_t* hist = reinterpret_cast<uint32_t*>(s.buf());
      s.clear();
      const float to_bin = SBINS / SRANGE;
      const float zmax = sample_dist(tmax, top, s.inv_t);
      const bool by_max = k && k <= p.ctas * S::NTH / 2;  // enough maxima to bound the k-th largest from below
      if (zmax < SRANGE) atomicAdd(&hist[min(SBINS - 1, static_cast<int>(zmax * to_bin))],
                                   k ? 1u : static_cast<uint32_t>(__expf(-zmax) * 131072.f));
      float spread = 0.f;  // the estimate's variance
      if (!by_max) {
        const int ns = max(1, p.per / 8);
        const float f = static_cast<float>(p.per) / ns;
        for (int it = 0; it < ns; ++it) {
          float v[VEC];
          s.vec(it, v);
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            const float z = sample_dist(v[e], top, s.inv_t);
            if (v[e] < tmax && z < SRANGE) {
              const float ez = f * __expf(-z);
              spread = fmaf(ez, ez, spread);
              atomicAdd(&hist[min(SBINS - 1, static_cast<int>(z * to_bin))],
                        static_cast<uint32_t>(k ? f + 0.5f : ez * 131072.f + 0.5f));
            }
          }
        }
      }
      s.agree();
      // thread t: bins 2t and 2t + 1 of the whole row, and what the bins up to them hold
      unsigned long long part[CTAS], h0 = 0, h1 = 0;
      s.read_all(tid, part);
#pragma unroll
      for (int r = 0; r < CTAS; ++r) {
        h0 += part[r] & 0xFFFFFFFFull;
        h1 += part[r] >> 32;
      }
      unsigned long long c = h0 + h1;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const unsigned long long t = __shfl_up_sync(0xffffffffu, c, d);
        if (lane >= d) c += t;
      }
      if (lane == 31) s_tmp[w] = c;
      if (STREAM) {
        spread = warp_sum(spread);
        if (lane == 0) s_tmp[SW + w] = __float_as_uint(spread);
      }
      if (tid == 0) s_tmp[2 * SW + 2] = s_tmp[2 * SW + 3] = SBINS;
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
        // the tail below the cut is sampled well: an error of the sum moves the cut by its share of 1 - p.
        // With 2048 thread maxima 0.05 was enough; with 512 the sampled terms tell their own spread.
        double room = 0.05;
        if (STREAM) {
          spread = 0.f;
          for (int i = 0; i < SW; ++i) spread += __uint_as_float(static_cast<uint32_t>(s_tmp[SW + i]));
          room = 0.02 + 3.0 * sqrtf(spread) * 131072.0 / (static_cast<double>(total) + 1.0);
        }
        const double q = fmax(static_cast<double>(tp), 0.0);
        room = room * (1.0 - q) + 1e-4;
        want_lo = (q + room) * total;
        want_hi = (q - room) * total;
      }
      if (c0 >= want_lo && b0 < want_lo) s_tmp[2 * SW + 2] = 2 * tid;
      else if (c >= want_lo && c0 < want_lo) s_tmp[2 * SW + 2] = 2 * tid + 1;
      if (b0 <= want_hi && c0 > want_hi) s_tmp[2 * SW + 3] = 2 * tid;
      else if (c0 <= want_hi && c > want_hi) s_tmp[2 * SW + 3] = 2 * tid + 1;
      __syncthreads();
      const int blo = static_cast<int>(s_tmp[2 * SW + 2]), bhi = static_cast<int>(s_tmp[2 * SW + 3]);
      __syncthreads();
      s.next();
      if (blo < SBINS) {
        const float e = top - (blo + (by_max ? 1 : 2)) / to_bin / s.inv_t;  // (a bin to spare)
        if (e == e) glo = max(low, min(Key::of(e), tk));
      }
      if (want_hi > 0 && bhi < SBINS && bhi > 0) {
        const float e = top - (bhi - 1) / to_bin / s.inv_t;
        if (e == e) ghi = min(high, max(Key::of(e), glo + 1));
      }
    }

    // tokens of key `cut` that stay when the weight above it is acc
    auto ties_of = [&](unsigned long long bound, unsigned long long acc) -> long long {
      const unsigned long long wt = s.weight_of(cut);
      return wt ? static_cast<long long>((bound - acc + wt - 1) / wt) : V;
    };
    unsigned long long bound = k, acc = 0;
    int found = S::NONE;
    bool whole_row = false;
    if (k) {
      found = s.template search<false>(low, high, glo, high, bound, false, cut, acc);
      if (found == S::CUT) ties = k - static_cast<long long>(acc);
    }
    if (nucleus && found == S::NONE) {
      // of the whole row (or of fewer than k tokens of any weight)
      whole_row = true;
      bound = fixed32(tp);
      found = s.template search<true>(low, high, k ? low : glo, k ? high : ghi, bound, true, cut, acc);
      if (found == S::CUT) ties = ties_of(bound, acc);
    } else if (nucleus && found == S::CUT) {
      // of the first k: their weight above the cut first
      unsigned long long v[1] = {0};
      const bool listed = s.list_ok && s.list_hi == high;
      if (listed) {
        for (int i = lane; i < s.n_list; i += 32)
          if (s.list[i].x > cut) v[0] += s.weight_of(s.list[i].x);
      } else {
        unsigned long long in_list, all;
        s.template pass<true>(cut, cut + 1, in_list, all);
        v[0] = s.above;
        s.list_ok = false;
      }
      s.sums(v);
      const unsigned long long sum = v[0];
      bound = max(1ull, scaled_ceil(sum + ties * s.weight_of(cut), fixed32(tp)));
      if (bound > sum) {
        ties = min(ties, ties_of(bound, sum));
      } else {
        acc = 0;
        if (listed) {
          cut = s.template radix<true>(cut + 1, acc, bound);
          ties = ties_of(bound, acc);
        } else {
          found = s.template search<true>(cut + 1, high, cut + 1, high, bound, false, cut, acc);
          if (found == S::CUT) ties = ties_of(bound, acc);
        }
      }
      if (found == S::FEW) {
        // every token of the bracket is in the lists and the bound is known: the cut from them
        acc = 0;
        cut = s.template radix<true>(cut + 1, acc, bound);
        ties = ties_of(bound, acc);
        found = S::CUT;
      }
    }
    if (found == S::FEW) {
      // gathered over CTA 0's slice: every pass over it has ended
      s.few(row, k, nucleus, tp, whole_row ? bound : 0, least,
            reinterpret_cast<uint4*>(smem + SW * SLIST * sizeof(uint2)));
      return;
    }
  }

  // ---- every warp's kept weight, number kept, and tokens of the cut's own key
  const float fcut = cut ? Key::value(cut) : -INFINITY;
  const uint32_t wt = cut ? sample_weight(fcut, top, s.inv_t) : 0u;
  if (wt < least) ties = 0;
  unsigned long long sum = 0;
  unsigned int n_kept = 0, n_tie = 0;
  // the list holds them all, or all that the last pass did not sum already
  const bool listed = s.list_ok && (s.list_hi == high ||
                                    (s.summed && sample_weight(Key::value(s.list_hi), top, s.inv_t) >= least));
  if (listed) {
    if (s.list_hi != high) {
      sum = s.above;
      n_kept = s.n_above;
    }
    for (int i = lane; i < s.n_list; i += 32) {
      const uint32_t key = s.list[i].x;
      const uint32_t wi = sample_weight(Key::value(key), top, s.inv_t);
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
  // lane l: chunks 2l and 2l + 1 of the row's ctas * SW
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

  s.next();
  s.agree();  // nobody reads this CTA's buffers any more
  // ---- the CTA whose chunk it is finds the token: warp i takes the chunk's i-th 256 (or 128) elements of every eight
  if (chunk / SW != s.rank) return;
  for (int it0 = 0; it0 < p.per; it0 += SW) {
    const int it = it0 + w;
    float v[VEC];
    if (it < p.per) {
      s.at(chunk % SW, it, v);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[e] = -INFINITY;
    }
    int nt = 0;
#pragma unroll
    for (int e = 0; e < VEC; ++e) nt += v[e] == fcut;
    int pre = nt;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int t = __shfl_up_sync(0xffffffffu, pre, d);
      if (lane >= d) pre += t;
    }
    __syncthreads();
    if (lane == 31) s_tmp[w] = pre;
    __syncthreads();
    long long rank = tie_run + pre - nt;
    for (int i = 0; i < SW; ++i) {
      const long long n = static_cast<long long>(s_tmp[i]);
      if (i < w) rank += n;
      tie_run += n;
    }
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
    if (lane == 31) s_tmp[SW + w] = end;
    __syncthreads();
    end += run;
    for (int i = 0; i < SW; ++i) {
      const unsigned long long n = s_tmp[SW + i];
      if (i < w) end += n;
      run += n;
    }
    if (end > target && end - mine <= target) {
      unsigned long long at = end - mine;
      int e = 0;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        at += we[i];
        if (at <= target) e = i + 1;
      }
      float xe = v[0];
#pragma unroll
      for (int i = 1; i < VEC; ++i)
        if (i == e) xe = v[i];
      s.finish(row, (chunk * p.per + it) * 32 * VEC + lane * VEC + e, xe, total, static_cast<int>(kept_all));
    }
    if (run > target) break;  // the same in every warp
  }
}

// CTAs per row and vectors per lane.  Slices of 32 KB leave room for four CTAs
// per SM, whose barriers and passes overlap; few rows are cut finer, down to
// one vector per lane, until there are two CTAs per SM.  Eight CTAs is the
// portable cluster size.
static void sample_shape(int rows, int V, int esize, int& ctas, int& per) {
  const int vec = 16 / esize, chunk = 256 * vec;  // elements per CTA and vector
  ctas = 1;
  while (ctas < SCTAS && (static_cast<long long>(V) * esize > static_cast<long long>(ctas) * 32768 ||
                          (static_cast<long long>(rows) * ctas * 2 <= 296 && V > ctas * chunk)))
    ctas *= 2;
  per = (V + ctas * chunk - 1) / (ctas * chunk);
}

template <typename T, bool STREAM>
static cudaError_t sample_launch(const SampleParams& p, cudaStream_t st) {
  using S = Sampler<T, STREAM>;
  // the widest slice: kSampleMaxV fp32 logits over SCTAS CTAs
  constexpr int lists = S::SW * S::SLIST * static_cast<int>(sizeof(uint2));
  cudaError_t e = allow_smem<sample_kernel<T, STREAM>>(lists + (STREAM ? SSMALL * 16 : kSampleMaxV / SCTAS * 4));
  if (e != cudaSuccess) return e;
  return launch_early(sample_kernel<T, STREAM>, dim3(static_cast<unsigned>(p.rows) * p.ctas), S::NTH,
                      lists + (STREAM ? SSMALL * sizeof(uint4) : static_cast<size_t>(p.per) * S::NTH * 16), st, p,
                      p.ctas);
}

// One CTA per row pays when rows are wide and there is one for every SM (us,
// cluster / one CTA, nucleus 0.9 and top-k 50): 64 KB rows 25 / 29 and 15 / 17 at
// 148 rows, 57 / 70 and 33 / 39 at 512; 128 KB rows 34 / 32 and 21 / 18 at 148,
// 100 / 88 and 56 / 43 at 512; 256 KB rows 83 / 84 and 52 / 40 at 148, 253 / 197
// and 158 / 95 at 512; 512 KB rows 136 / 107 and 76 / 56 at 148, 435 / 262 and
// 231 / 135 at 512.
template <typename T>
static cudaError_t sample_t(SampleParams p, cudaStream_t st) {
  sample_shape(p.rows, p.V, sizeof(T), p.ctas, p.per);
  if (static_cast<long long>(p.V) * sizeof(T) > 65536 && p.rows >= 148) {
    constexpr int chunk = Sampler<T, true>::NTH * Sampler<T, true>::VEC;
    p.ctas = 1;
    p.per = (p.V + chunk - 1) / chunk;
    return sample_launch<T, true>(p, st);
  }
  return sample_launch<T, false>(p, st);
}

}  // namespace tkb
