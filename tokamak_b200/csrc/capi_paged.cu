// capi_paged.cu -- extern "C" entry points of the paged key-value cache and of
// sampling (include/tkm_b200.h).  Compiled in the same translation unit as
// capi.cu and capi_rows.cu (tkb_all.cu).

namespace {

constexpr int kMaxSeqs = 4096;  // sequences per cache: their tile counts are scanned in shared memory

int dtype_bytes(int dt) { return dt == TKB_F32 ? 4 : 2; }

int cache_check(const char* who, const tkb_kv_cache* c) {
  if (!c) return fail(TKB_ERR_ARG, "%s: null cache", who);
  if (!dtype_ok(c->dtype)) return fail(TKB_ERR_ARG, "%s: bad dtype %d", who, c->dtype);
  if (c->B <= 0 || c->Hkv <= 0 || c->n_pages <= 0 || c->max_pages <= 0)
    return fail(TKB_ERR_ARG, "%s: B, Hkv, n_pages and max_pages must be positive", who);
  if (c->B > kMaxSeqs) return fail(TKB_ERR_UNSUPPORTED, "%s: B %d > %d", who, c->B, kMaxSeqs);
  if (c->D != 64 && c->D != 128) return fail(TKB_ERR_UNSUPPORTED, "%s: head dim %d not in {64, 128}", who, c->D);
  if (c->page_size <= 0 || c->page_size % 16 || c->page_size > 1024)
    return fail(TKB_ERR_ARG, "%s: page_size %d is not a multiple of 16 up to 1024", who, c->page_size);
  if (static_cast<long long>(c->max_pages) * c->page_size > 0x3FFFFFFF)
    return fail(TKB_ERR_ARG, "%s: max_pages * page_size above 2^30 - 1", who);
  if (!c->k || !c->v || !c->block_table || !c->seq_lens) return fail(TKB_ERR_ARG, "%s: null pointer in the cache", who);
  if (!aligned16(c->k) || !aligned16(c->v)) return fail(TKB_ERR_ARG, "%s: k and v must be 16-byte aligned", who);
  if (c->page_stride < static_cast<long long>(c->Hkv) * c->page_size * c->D ||
      c->page_stride * dtype_bytes(c->dtype) % 16)
    return fail(TKB_ERR_ARG, "%s: page_stride %lld must hold Hkv * page_size * D elements and be a multiple of 16 bytes",
                who, c->page_stride);
  return TKB_OK;
}

// Rows of `width` elements, `stride` apart, moved in 16-byte vectors.
int rows_check(const char* who, const char* name, const void* p, long long stride, long long width, int dtype) {
  if (stride < width || stride * dtype_bytes(dtype) % 16 || !aligned16(p))
    return fail(TKB_ERR_ARG, "%s: %s must be 16-byte aligned rows at least %lld elements apart", who, name, width);
  return TKB_OK;
}

}  // namespace

extern "C" {

int tkb_kv_lens(int32_t* seq_lens, int32_t* seen, const int32_t* row_start, int add, int limit, int B, void* stream) {
  if (!seq_lens || B <= 0 || limit < 0 || add < 0) return fail(TKB_ERR_ARG, "tkb_kv_lens: bad arguments");
  kv_lens_kernel<<<(B + 255) / 256, 256, 0, static_cast<cudaStream_t>(stream)>>>(seq_lens, seen, row_start, add, limit,
                                                                               B);
  return cuda_status(cudaGetLastError(), "tkb_kv_lens", 1);
}

int tkb_kv_append(const tkb_kv_cache* cache, const void* qkv, long long qkv_stride, const float* bias,
                  const float* qk_gain, void* out, long long out_stride, int out_full, const int32_t* row_start,
                  const int32_t* seen, int rows, int Hq, int has_qknorm, int has_rope, float theta, float rope_scale,
                  float low_ff, float high_ff, float octx, void* stream) {
  const char* who = "tkb_kv_append";
  int rc = cache_check(who, cache);
  if (rc) return rc;
  if (rows <= 0 || Hq <= 0) return fail(TKB_ERR_ARG, "%s: rows and Hq must be positive", who);
  if (!row_start && rows != cache->B)
    return fail(TKB_ERR_ARG, "%s: without row_start there is one row per sequence (%d rows, B %d)", who, rows, cache->B);
  if (!qkv) return fail(TKB_ERR_ARG, "%s: null qkv", who);
  const long long C = static_cast<long long>(Hq + 2 * cache->Hkv) * cache->D;
  if (C > 0x3FFFFFFF) return fail(TKB_ERR_ARG, "%s: row of %lld columns", who, C);
  if ((rc = rows_check(who, "qkv", qkv, qkv_stride, C, cache->dtype))) return rc;
  if (out && (rc = rows_check(who, "out", out, out_stride, out_full ? C : static_cast<long long>(Hq) * cache->D,
                              cache->dtype)))
    return rc;
  if ((bias && !aligned16(bias)) || (qk_gain && !aligned16(qk_gain)))
    return fail(TKB_ERR_ARG, "%s: bias and qk_gain must be 16-byte aligned", who);
  if (has_rope && !(theta > 0.f)) return fail(TKB_ERR_ARG, "%s: theta must be positive", who);
  AppendParams p;
  memset(&p, 0, sizeof(p));
  p.c = *cache;
  p.qkv = qkv;
  p.qkv_stride = qkv_stride;
  p.bias = bias;
  p.gain = qk_gain;
  p.out = out;
  p.out_stride = out_stride;
  p.out_full = out_full ? 1 : 0;
  p.row_start = row_start;
  p.seen = seen;
  p.rows = rows;
  p.Hq = Hq;
  p.qknorm = has_qknorm ? 1 : 0;
  p.rope = has_rope ? 1 : 0;
  if (has_rope) p.tab = rope_table(cache->D, theta, rope_scale, low_ff, high_ff, octx);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
#define CALL(T) kv_append_t<T>(p, st)
  return cuda_status(TKB_BY_DTYPE(cache->dtype, CALL), who, 1);
#undef CALL
}

size_t tkb_paged_attn_decode_workspace(const tkb_kv_cache* cache, int Hq, int accumulate) {
  if (cache_check("tkb_paged_attn_decode_workspace", cache)) return 0;
  if (Hq <= 0 || Hq % cache->Hkv) {
    fail(TKB_ERR_ARG, "tkb_paged_attn_decode_workspace: Hq (%d) must be a multiple of Hkv (%d)", Hq, cache->Hkv);
    return 0;
  }
  return decode_ws(*cache, Hq, accumulate).bytes;
}

int tkb_paged_attn_decode(const tkb_kv_cache* cache, const void* q, long long q_stride, void* out,
                          long long out_stride, float* lse, int Hq, float scale, int accumulate, void* workspace,
                          size_t workspace_bytes, void* stream) {
  const char* who = "tkb_paged_attn_decode";
  int rc = cache_check(who, cache);
  if (rc) return rc;
  if (Hq <= 0 || Hq % cache->Hkv)
    return fail(TKB_ERR_ARG, "%s: Hq (%d) must be a multiple of Hkv (%d)", who, Hq, cache->Hkv);
  if (!q || !out) return fail(TKB_ERR_ARG, "%s: null pointer", who);
  const long long width = static_cast<long long>(Hq) * cache->D;
  if (width > 0x3FFFFFFF) return fail(TKB_ERR_ARG, "%s: row of %lld columns", who, width);
  if ((rc = rows_check(who, "q", q, q_stride, width, cache->dtype))) return rc;
  if ((rc = rows_check(who, "out", out, out_stride, width, cache->dtype))) return rc;
  if (accumulate && (!cache->weight || !aligned16(cache->weight)))
    return fail(TKB_ERR_ARG, "%s: accumulate needs the cache's weight, 16-byte aligned", who);
  if (static_cast<long long>(cache->B) * cache->Hkv > 65535)
    return fail(TKB_ERR_UNSUPPORTED, "%s: B * Hkv above 65535", who);
  if (static_cast<double>(cache->B) * Hq * cache->max_pages * cache->page_size > 8.0 * 0x3FFFFFFF)
    return fail(TKB_ERR_UNSUPPORTED, "%s: B * Hq * max_pages * page_size above 2^33", who);
  const size_t need = tkb_paged_attn_decode_workspace(cache, Hq, accumulate);
  if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255))
    return fail(TKB_ERR_WORKSPACE, "%s: workspace of %zu bytes, 256-byte aligned, required", who, need);
  DecodeParams p;
  memset(&p, 0, sizeof(p));
  p.c = *cache;
  p.q = q;
  p.q_stride = q_stride;
  p.out = out;
  p.out_stride = out_stride;
  p.lse = lse;
  p.Hq = Hq;
  p.G = Hq / cache->Hkv;
  p.qblocks = (p.G + QT - 1) / QT;
  p.accumulate = accumulate ? 1 : 0;
  p.scale_log2 = scale * 1.4426950408889634f;
  const DecodeWs w = decode_ws(*cache, Hq, accumulate);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  p.counters = reinterpret_cast<int*>(ws + w.counters);
  p.part = reinterpret_cast<float*>(ws + w.part);
  p.head = reinterpret_cast<float*>(ws + w.head);
  p.lse2 = reinterpret_cast<float*>(ws + w.lse2);
  p.scores = reinterpret_cast<float*>(ws + w.scores);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
#define CALL(T) paged_decode_t<T>(p, st)
  return cuda_status(TKB_BY_DTYPE(cache->dtype, CALL), who, accumulate ? 2 : 1);
#undef CALL
}

size_t tkb_kv_evict_workspace(const tkb_kv_cache* cache) {
  if (cache_check("tkb_kv_evict_workspace", cache)) return 0;
  return round256(evict_ws(*cache).bytes);
}

int tkb_kv_evict(const tkb_kv_cache* cache, const int32_t* seen, int budget, int recent, int sinks, void* workspace,
                 size_t workspace_bytes, void* stream) {
  const char* who = "tkb_kv_evict";
  int rc = cache_check(who, cache);
  if (rc) return rc;
  if (!seen || !cache->pos || !cache->weight)
    return fail(TKB_ERR_ARG, "%s: seen and the cache's pos and weight are needed", who);
  if (!aligned16(cache->pos) || !aligned16(cache->weight))
    return fail(TKB_ERR_ARG, "%s: pos and weight must be 16-byte aligned", who);
  if (budget <= 0 || recent < 0 || sinks < 0 || static_cast<long long>(recent) + sinks > budget)
    return fail(TKB_ERR_ARG, "%s: budget must be positive and hold recent + sinks tokens", who);
  const size_t need = tkb_kv_evict_workspace(cache);
  if (!workspace || workspace_bytes < need || !aligned16(workspace))
    return fail(TKB_ERR_WORKSPACE, "%s: workspace of %zu bytes, 16-byte aligned, required", who, need);
  EvictParams p;
  memset(&p, 0, sizeof(p));
  p.c = *cache;
  p.seen = seen;
  const EvictWs w = evict_ws(*cache);
  p.lists = static_cast<uint2*>(workspace);
  if (w.bytes > w.keys) p.keys = reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(workspace) + w.keys);
  p.budget = budget;
  p.recent = recent;
  p.sinks = sinks;
  p.cap = w.cap;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
#define CALL(T) kv_evict_t<T>(p, st)
  return cuda_status(TKB_BY_DTYPE(cache->dtype, CALL), who, 1);
#undef CALL
}

int tkb_sample_logits(const void* logits, long long ld, const float* u, const float* temperature,
                      const int32_t* top_k, const float* top_p, const float* min_p, int32_t* token, float* logprob,
                      int32_t* kept, int rows, int V, int dtype, void* stream) {
  const char* who = "tkb_sample_logits";
  if (rows <= 0 || V <= 0) return fail(TKB_ERR_ARG, "%s: rows and V must be positive", who);
  if (V > kSampleMaxV) return fail(TKB_ERR_UNSUPPORTED, "%s: V %d > 2^18", who, V);
  if (rows > (1 << 26)) return fail(TKB_ERR_UNSUPPORTED, "%s: %d rows > 2^26", who, rows);
  if (!dtype_ok(dtype)) return fail(TKB_ERR_ARG, "%s: bad dtype %d", who, dtype);
  if (!logits || !u || !token) return fail(TKB_ERR_ARG, "%s: null pointer", who);
  if (ld < V) return fail(TKB_ERR_ARG, "%s: ld %lld < V %d", who, ld, V);
  if (reinterpret_cast<uintptr_t>(logits) % dtype_bytes(dtype))
    return fail(TKB_ERR_ARG, "%s: logits not aligned to their type", who);
  const SampleParams p = {logits, ld, u, temperature, top_k, top_p, min_p, token, logprob, kept, rows, V, 0, 0};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
#define CALL(T) sample_t<T>(p, st)
  return cuda_status(TKB_BY_DTYPE(dtype, CALL), who, 1);
#undef CALL
}

}  // extern "C"
