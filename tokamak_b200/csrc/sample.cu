// sample.cu -- one token per row of logits from given uniform numbers:
// temperature, top-k, top-p (nucleus), min-p.
//
// Every token's weight exp(-(max - x)/T) is a whole multiple of 2^-31, so its
// sums are exact 64-bit integers (V <= 2^20 keeps them below 2^51) and the
// token cannot depend on how a sum is cut over threads.  All three
// truncations keep a prefix of the order "falling logit, equal ones by
// index", so a row's kept set is described by a key, the number of tokens of
// exactly that key that stay, and a least weight.
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
};

constexpr int SNT = 1024;

TKB_DEVFN unsigned long long block_sum_u64(unsigned long long v, unsigned long long* sh) {
#pragma unroll
  for (int m = 16; m >= 1; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
  __syncthreads();
  if (lane_id() == 0) sh[warp_id()] = v;
  __syncthreads();
  unsigned long long s = 0;
  for (int i = 0; i < SNT / 32; ++i) s += sh[i];
  return s;
}

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
// The whole weight of logit x in a row of maximum `top`.
TKB_DEVFN uint32_t sample_weight(float x, float top, float inv_t) {
  const float z = x == top ? 0.f : __fmul_rn(__fsub_rn(top, x), inv_t);
  return __float2uint_rn(expf(-z) * 2147483648.f);
}

template <typename T>
__global__ void __launch_bounds__(SNT) sample_kernel(const __grid_constant__ SampleParams p) {
  __shared__ unsigned long long sh[SNT / 32];
  __shared__ float sh_f[SNT / 32];
  __shared__ int sh_i[SNT / 32];
  __shared__ int s_token;
  __shared__ float s_x;
  const int row = blockIdx.x, tid = threadIdx.x, V = p.V;
  const T* x = static_cast<const T*>(p.logits) + row * p.ld;
  auto logit = [&](int i) {
    const float v = Elem<T>::ld(x + i);
    return v != v ? -INFINITY : v;
  };
  float top = -INFINITY;
  for (int i = tid; i < V; i += SNT) top = fmaxf(top, logit(i));
  top = warp_max(top);
  if (lane_id() == 0) sh_f[warp_id()] = top;
  __syncthreads();
  for (int i = 0; i < SNT / 32; ++i) top = fmaxf(top, sh_f[i]);
  if (tid == 0) s_token = -1;
  const float temp = p.temperature ? p.temperature[row] : 1.f;
  const bool greedy = !(temp > 0.f);
  const float inv_t = greedy ? 1.f : __frcp_rn(temp);
  if (top == -INFINITY) {
    if (tid == 0) {
      p.token[row] = -1;
      if (p.logprob) p.logprob[row] = -INFINITY;
      if (p.kept) p.kept[row] = 0;
    }
    return;
  }
  auto weight = [&](float v) { return sample_weight(v, top, inv_t); };

  // kept: key > cut, and the first `ties` tokens of key == cut
  uint32_t cut = 0;
  int ties = V;
  const int k = greedy ? 1 : (p.top_k && p.top_k[row] > 0 ? p.top_k[row] : V);
  if (k < V) {
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t next = cut | (1u << bit);
      unsigned long long n = 0;
      for (int i = tid; i < V; i += SNT) n += order_key(logit(i)) >= next;
      if (block_sum_u64(n, sh) >= k) cut = next;
    }
    unsigned long long n = 0;
    for (int i = tid; i < V; i += SNT) n += order_key(logit(i)) > cut;
    ties = k - static_cast<int>(block_sum_u64(n, sh));
  }
  const float tp = p.top_p ? p.top_p[row] : 1.f;
  if (!greedy && !(tp >= 1.f)) {
    const unsigned long long part = fixed32(tp);
    // weight of the tokens above a key (within the first k)
    auto above = [&](uint32_t key, bool equal) {
      unsigned long long w = 0;
      for (int i = tid; i < V; i += SNT) {
        const float v = logit(i);
        const uint32_t o = order_key(v);
        if (o > key || (equal && o == key)) w += weight(v);
      }
      return block_sum_u64(w, sh);
    };
    auto tie_weight = [&](uint32_t key) -> unsigned long long {
      // key back to its float
      const uint32_t u = key & 0x80000000u ? key & 0x7FFFFFFFu : ~key;
      const float v = __uint_as_float(u);
      return key == 0 ? 0 : weight(v);
    };
    unsigned long long total;
    if (k < V) total = above(cut, false) + static_cast<unsigned long long>(ties) * tie_weight(cut);
    else total = above(0, true);
    const unsigned long long bound = scaled_ceil(total, part);
    uint32_t key = cut;
    if (above(cut, false) < bound) {
      // the bound falls among the ties of the cut itself
      const unsigned long long w = tie_weight(cut), a = above(cut, false);
      if (w) {
        const unsigned long long t = (bound - a + w - 1) / w;
        if (t < static_cast<unsigned long long>(ties)) ties = static_cast<int>(t);
      }
    } else {
      // the largest key whose tokens, with all above, reach the bound
      key = 0;
      for (int bit = 31; bit >= 0; --bit) {
        const uint32_t next = key | (1u << bit);
        if (above(next, true) >= bound) key = next;
      }
      const unsigned long long w = tie_weight(key), a = above(key, false);
      unsigned long long t = w ? (bound > a ? (bound - a + w - 1) / w : 0) : 0;
      if (a == 0 && t == 0) {
        t = 1;
        key = order_key(top);  // bound 0: the first token alone
      }
      cut = key;
      ties = static_cast<int>(t < static_cast<unsigned long long>(V) ? t : V);
    }
  }
  uint32_t least = 1;
  if (!greedy && p.min_p && p.min_p[row] > 0.f)
    least = p.min_p[row] >= 1.f ? 0x80000000u : static_cast<uint32_t>(ceil(static_cast<double>(p.min_p[row]) * 2147483648.0));
  if (least < 1) least = 1;

  // total of the kept weights, then the token where the running sum passes u * total
  unsigned long long total = 0, target = 0;
  int n_kept = 0;
  for (int pass = 0; pass < 2; ++pass) {
    unsigned long long run = 0;
    int tie_run = 0;
    for (int i0 = 0; i0 < V; i0 += SNT) {
      const int i = i0 + tid;
      const float v = i < V ? logit(i) : -INFINITY;
      const uint32_t o = i < V ? order_key(v) : 0u;
      const bool tie = i < V && o == cut;
      int tot;
      const int rank = tie_run + block_scan(tie, sh_i, tot) - tie;
      tie_run += tot;
      const uint32_t w0 = i < V ? weight(v) : 0u;
      const bool keep = i < V && w0 >= least && (o > cut || (tie && rank < ties));
      const unsigned long long w = keep ? w0 : 0u;
      if (pass == 0) {
        total += w;
        n_kept += keep;
        continue;
      }
      // inclusive prefix over the block
      unsigned long long s = w;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const unsigned long long t = __shfl_up_sync(0xffffffffu, s, d);
        if (lane_id() >= d) s += t;
      }
      __syncthreads();
      if (lane_id() == 31) sh[warp_id()] = s;
      __syncthreads();
      unsigned long long all = 0;
      for (int j = 0; j < SNT / 32; ++j) {
        if (j < warp_id()) s += sh[j];
        all += sh[j];
      }
      s += run;
      if (keep && s > target && s - w <= target) {
        s_token = i;
        s_x = v;
      }
      run += all;
    }
    if (pass == 0) {
      total = block_sum_u64(total, sh);
      n_kept = static_cast<int>(block_sum_u64(n_kept, sh));
      target = scaled_floor(total, fixed32(p.u[row]));
    }
  }
  __syncthreads();
  if (tid == 0) {
    p.token[row] = s_token;
    if (p.kept) p.kept[row] = n_kept;
    const float z = s_x == top ? 0.f : (top - s_x) * inv_t;
    if (p.logprob) p.logprob[row] = greedy ? 0.f : -z - logf(static_cast<float>(total) * 4.656612873077393e-10f);
  }
}

template <typename T>
static cudaError_t sample_t(const SampleParams& p, cudaStream_t st) {
  sample_kernel<T><<<p.rows, SNT, 0, st>>>(p);
  return cudaGetLastError();
}

}  // namespace tkb
