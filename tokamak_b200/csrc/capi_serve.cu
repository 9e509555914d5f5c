// capi_serve.cu -- extern "C" entry points of the operators that serve many
// requests at once (include/tkm_b200.h).  Compiled in the same translation
// unit as capi_paged.cu (tkb_all.cu), whose checks it uses.

namespace {

// The sequences' rows: row_start, or one row each.
int batch_check(const char* who, const void* row_start, int rows, int B) {
  if (rows <= 0 || B <= 0) return fail(TKB_ERR_ARG, "%s: rows and B must be positive", who);
  if (B > kMaxSeqs) return fail(TKB_ERR_UNSUPPORTED, "%s: B %d > %d", who, B, kMaxSeqs);
  if (rows > (1 << 26)) return fail(TKB_ERR_UNSUPPORTED, "%s: %d rows > 2^26", who, rows);
  if (!row_start && rows != B)
    return fail(TKB_ERR_ARG, "%s: without row_start there is one row per sequence (%d rows, B %d)", who, rows, B);
  return TKB_OK;
}

constexpr int kLoraRows = 1 << 21;  // rows of a plan: its tiles are counted in a grid's second dimension
int lora_check(const char* who, const void* row_start, int rows, int B, int n_adapters) {
  int rc = batch_check(who, row_start, rows, B);
  if (rc) return rc;
  if (n_adapters <= 0) return fail(TKB_ERR_ARG, "%s: n_adapters must be positive", who);
  if (rows > kLoraRows) return fail(TKB_ERR_UNSUPPORTED, "%s: %d rows > 2^21", who, rows);
  return TKB_OK;
}

int chunk_check(const char* who, const tkb_kv_cache* c, int rows, int Hq) {
  int rc = cache_check(who, c);
  if (rc) return rc;
  if (Hq <= 0 || Hq % c->Hkv) return fail(TKB_ERR_ARG, "%s: Hq (%d) must be a multiple of Hkv (%d)", who, Hq, c->Hkv);
  if (static_cast<long long>(Hq) * c->D > 0x3FFFFFFF) return fail(TKB_ERR_ARG, "%s: row of %d heads", who, Hq);
  return batch_check(who, c, rows, c->B);
}

}  // namespace

extern "C" {

size_t tkb_paged_attn_chunk_workspace(const tkb_kv_cache* cache, int rows, int Hq) {
  if (chunk_check("tkb_paged_attn_chunk_workspace", cache, rows, Hq)) return 0;
  return round256(chunk_ws(*cache).bytes);
}

int tkb_paged_attn_chunk(const tkb_kv_cache* cache, const void* q, long long q_stride, void* out,
                         long long out_stride, float* lse, const int32_t* row_start, int rows, int Hq, float scale,
                         void* workspace, size_t workspace_bytes, void* stream) {
  const char* who = "tkb_paged_attn_chunk";
  int rc = chunk_check(who, cache, rows, Hq);
  if (rc) return rc;
  if ((rc = batch_check(who, row_start, rows, cache->B))) return rc;
  if (!q || !out) return fail(TKB_ERR_ARG, "%s: null pointer", who);
  if (!(scale > 0.f) || std::isinf(scale)) return fail(TKB_ERR_ARG, "%s: scale must be positive", who);
  const long long width = static_cast<long long>(Hq) * cache->D;
  // the units' costs are summed in 64 bits
  if (static_cast<double>(rows) * Hq * cache->max_pages * cache->page_size > 9e15)
    return fail(TKB_ERR_UNSUPPORTED, "%s: rows * Hq * max_pages * page_size above 9e15", who);
  if ((rc = rows_check(who, "q", q, q_stride, width, cache->dtype))) return rc;
  if ((rc = rows_check(who, "out", out, out_stride, width, cache->dtype))) return rc;
  const size_t need = tkb_paged_attn_chunk_workspace(cache, rows, Hq);
  if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255))
    return fail(TKB_ERR_WORKSPACE, "%s: workspace of %zu bytes, 256-byte aligned, required", who, need);
  ChunkParams p;
  memset(&p, 0, sizeof(p));
  p.c = *cache;
  p.q = q;
  p.q_stride = q_stride;
  p.out = out;
  p.out_stride = out_stride;
  p.lse = lse;
  p.row_start = row_start;
  p.rows = rows;
  p.Hq = Hq;
  p.G = Hq / cache->Hkv;
  p.scale_log2 = scale * 1.4426950408889634f;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
#define CALL(T) paged_chunk_t<T>(p, workspace, st)
  return cuda_status(TKB_BY_DTYPE(cache->dtype, CALL), who, 2);
#undef CALL
}

int tkb_kv_pages(int32_t* block_table, int32_t* held, const int32_t* lens, int32_t* free_pages, int32_t* n_free,
                 int32_t* granted, int64_t* slots, const int32_t* row_start, int rows, int B, int max_pages,
                 int page_size, int n_pages, void* stream) {
  const char* who = "tkb_kv_pages";
  if (!block_table || !held || !lens || !free_pages || !n_free) return fail(TKB_ERR_ARG, "%s: null pointer", who);
  int rc = batch_check(who, slots ? static_cast<const void*>(row_start) : block_table, slots ? rows : 1, B);
  if (rc) return rc;
  if (max_pages <= 0 || n_pages <= 0) return fail(TKB_ERR_ARG, "%s: max_pages and n_pages must be positive", who);
  if (page_size <= 0 || page_size > 1024) return fail(TKB_ERR_ARG, "%s: page_size %d is not in 1 to 1024", who, page_size);
  if (static_cast<long long>(B) * max_pages >= (1 << 30) || n_pages >= (1 << 30))
    return fail(TKB_ERR_UNSUPPORTED, "%s: B * max_pages or n_pages above 2^30", who);
  if (reinterpret_cast<uintptr_t>(slots) & 7) return fail(TKB_ERR_ARG, "%s: slots must be 8-byte aligned", who);
  const PagesParams p = {block_table, held, lens, free_pages, n_free, granted, reinterpret_cast<long long*>(slots),
                         row_start, rows > 0 ? rows : 0, B, max_pages, page_size, n_pages};
  unsigned kernels = 0;
  const cudaError_t e = kv_pages(p, static_cast<cudaStream_t>(stream), kernels);
  return cuda_status(e, who, kernels);
}

size_t tkb_lora_plan_bytes(int B, int rows, int n_adapters) {
  const char* who = "tkb_lora_plan_bytes";
  if (lora_check(who, who, rows, B, n_adapters)) return 0;
  return lora_plan_at(B, rows, n_adapters).bytes;
}

int tkb_lora_plan(const int32_t* adapter, const int32_t* row_start, int B, int rows, int n_adapters, void* plan,
                  size_t plan_bytes, void* stream) {
  const char* who = "tkb_lora_plan";
  int rc = lora_check(who, row_start, rows, B, n_adapters);
  if (rc) return rc;
  if (!adapter) return fail(TKB_ERR_ARG, "%s: null pointer", who);
  const size_t need = tkb_lora_plan_bytes(B, rows, n_adapters);
  if (!plan || plan_bytes < need || (reinterpret_cast<uintptr_t>(plan) & 255))
    return fail(TKB_ERR_WORKSPACE, "%s: plan of %zu bytes, 256-byte aligned, required", who, need);
  const LoraPlanAt at = lora_plan_at(B, rows, n_adapters);
  uint8_t* base = static_cast<uint8_t*>(plan);
  const LoraPlanParams p = {adapter, row_start, static_cast<int*>(plan), reinterpret_cast<LoraTile*>(base + 256),
                            reinterpret_cast<int32_t*>(base + at.rows), B, rows, n_adapters, at.tm, 0};
  return cuda_status(lora_plan(p, at.tiles * at.tm, static_cast<cudaStream_t>(stream)), who, 1);
}

size_t tkb_lora_workspace(int rows, int R) {
  if (rows <= 0 || rows > kLoraRows || R <= 0 || R > 128) {
    fail(TKB_ERR_ARG, "tkb_lora_workspace: rows are 1 to 2^21, R 1 to 128");
    return 0;
  }
  return round256(static_cast<size_t>(rows) * lora_rank(R) * 4);
}

int tkb_lora_add(const void* plan, const void* x, long long x_stride, const void* A, const void* B_, const float* scale,
                 const void* y, long long y_stride, void* out, long long out_stride, int B, int rows, int n_adapters,
                 int K, int N, int R, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  const char* who = "tkb_lora_add";
  if (!plan || !x || !A || !B_ || !y || !out) return fail(TKB_ERR_ARG, "%s: null pointer", who);
  int rc = lora_check(who, plan, rows, B, n_adapters);
  if (rc) return rc;
  if (!dtype_ok(dtype)) return fail(TKB_ERR_ARG, "%s: bad dtype %d", who, dtype);
  if (K <= 0 || N <= 0) return fail(TKB_ERR_ARG, "%s: K and N must be positive", who);
  if (R <= 0 || R % 8 || R > 128) return fail(TKB_ERR_UNSUPPORTED, "%s: rank %d is not a multiple of 8 up to 128", who, R);
  const int e = dtype_bytes(dtype);
  if (static_cast<long long>(K) * e % 16 || static_cast<long long>(N) * e % 16 || K > (1 << 26) || N > (1 << 26))
    return fail(TKB_ERR_ARG, "%s: K and N must be multiples of 16 bytes", who);
  if ((rc = rows_check(who, "x", x, x_stride, K, dtype)) || (rc = rows_check(who, "y", y, y_stride, N, dtype)) ||
      (rc = rows_check(who, "out", out, out_stride, N, dtype)))
    return rc;
  if (y == out && y_stride != out_stride) return fail(TKB_ERR_ARG, "%s: out is y at another stride", who);
  if (!aligned16(A) || !aligned16(B_)) return fail(TKB_ERR_ARG, "%s: A and B must be 16-byte aligned", who);
  const size_t need = tkb_lora_workspace(rows, R);
  if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255))
    return fail(TKB_ERR_WORKSPACE, "%s: workspace of %zu bytes, 256-byte aligned, required", who, need);
  const LoraPlanAt at = lora_plan_at(B, rows, n_adapters);
  const uint8_t* base = static_cast<const uint8_t*>(plan);
  LoraParams p;
  memset(&p, 0, sizeof(p));
  p.n_tiles = static_cast<const int*>(plan);
  p.tiles = reinterpret_cast<const LoraTile*>(base + 256);
  p.row_of = reinterpret_cast<const int32_t*>(base + at.rows);
  p.x = x;
  p.a = A;
  p.b = B_;
  p.y = y;
  p.out = out;
  p.scale = scale;
  p.t = static_cast<float*>(workspace);
  p.x_stride = x_stride;
  p.y_stride = y_stride;
  p.out_stride = out_stride;
  p.rows = rows;
  p.K = K;
  p.N = N;
  p.R = R;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  unsigned kernels = 0;
#define CALL(T) lora_add_t<T>(p, at, st, kernels)
  const cudaError_t status = TKB_BY_DTYPE(dtype, CALL);
#undef CALL
  return cuda_status(status, who, kernels);
}

}  // extern "C"
