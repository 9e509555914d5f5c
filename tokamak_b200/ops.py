"""Torch-tensor wrappers over the C ABI (include/tkm_b200.h).

Each function allocates its outputs with torch on the tensors' device, calls
the corresponding ``tkb_*`` entry point on the current CUDA stream and raises
``TkbError`` on any failure.  No computation happens in Python.
"""
import ctypes

import torch

from . import DTYPE_BF16, DTYPE_F16, DTYPE_F32, TkbError, check, lib

_DT = {torch.float32: DTYPE_F32, torch.bfloat16: DTYPE_BF16, torch.float16: DTYPE_F16}


def dtype_code(t):
    try:
        return _DT[t.dtype]
    except KeyError:
        raise TkbError(f"unsupported dtype {t.dtype}")


def _p(t):
    return ctypes.c_void_p(t.data_ptr()) if t is not None else None


def _stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def _ws(nbytes, device):
    if nbytes == 0:
        return None, 0
    return torch.empty(nbytes, dtype=torch.uint8, device=device), nbytes


def gqa_attn_fwd(qkv, B, S, Hq, Hkv, D, scale=None, causal=True):
    """qkv: [B, S, (Hq+2Hkv)*D] -> (out [B, S, Hq*D], lse [B*Hq, S] fp32)."""
    scale = D ** -0.5 if scale is None else scale
    out = torch.empty(B, S, Hq * D, dtype=qkv.dtype, device=qkv.device)
    lse = torch.empty(B * Hq, S, dtype=torch.float32, device=qkv.device)
    check(lib().tkb_gqa_attn_fwd(_p(qkv), _p(out), _p(lse), B, S, Hq, Hkv, D, scale, int(causal),
                                 dtype_code(qkv), _stream()), "tkb_gqa_attn_fwd")
    return out, lse


def gqa_attn_bwd(qkv, out, dout, lse, B, S, Hq, Hkv, D, scale=None, causal=True, workspace=None, dqkv=None,
                 keep_ds=True):
    """keep_ds: offer the workspace that stores dS (dQ as a GEMM over it);
    False gives the minimum workspace, on which dQ recomputes S, P and dP."""
    scale = D ** -0.5 if scale is None else scale
    L = lib()
    dt = dtype_code(qkv)
    if keep_ds:
        need = L.tkb_gqa_attn_bwd_workspace_ex(B, S, Hq, D, int(causal), dt)
    else:
        need = L.tkb_gqa_attn_bwd_workspace(B, S, Hq, D, dt)
    if workspace is None:
        workspace, _ = _ws(need, qkv.device)
    else:
        need = workspace.numel() * workspace.element_size()
    if dqkv is None:
        dqkv = torch.empty_like(qkv)
    check(L.tkb_gqa_attn_bwd(_p(qkv), _p(out), _p(dout), _p(lse), _p(dqkv), _p(workspace), need, B, S, Hq, Hkv,
                             D, scale, int(causal), dt, _stream()), "tkb_gqa_attn_bwd")
    return dqkv


def add_rmsnorm_fwd(x, r, gamma, eps=1e-5):
    rows, C = x.shape[0], x.shape[-1]
    s = torch.empty_like(x) if r is not None else None
    y = torch.empty_like(x)
    istd = torch.empty(rows, dtype=torch.float32, device=x.device)
    check(lib().tkb_add_rmsnorm_fwd(_p(x), _p(r), _p(s), _p(y), _p(gamma), _p(istd), rows, C, eps,
                                    dtype_code(x), _stream()), "tkb_add_rmsnorm_fwd")
    return (s if s is not None else x), y, istd


def add_rmsnorm_bwd(dy, s, gamma, istd, ds_skip=None, dgamma=None):
    rows, C = s.shape[0], s.shape[-1]
    L = lib()
    dx = torch.empty_like(s)
    need = L.tkb_add_rmsnorm_bwd_workspace(rows, C)
    ws, _ = _ws(need, s.device)
    check(L.tkb_add_rmsnorm_bwd(_p(dy), _p(s), _p(gamma), _p(istd), _p(ds_skip), _p(dx), _p(dgamma), _p(ws),
                                need, rows, C, dtype_code(s), _stream()), "tkb_add_rmsnorm_bwd")
    return dx


def swiglu_fwd(gu, bg=None, bu=None):
    rows, F = gu.shape[0], gu.shape[-1] // 2
    h = torch.empty(rows, F, dtype=gu.dtype, device=gu.device)
    check(lib().tkb_swiglu_fwd(_p(gu), _p(bg), _p(bu), _p(h), rows, F, dtype_code(gu), _stream()),
          "tkb_swiglu_fwd")
    return h


def swiglu_bwd(dh, gu, bg=None, bu=None, dbg=None, dbu=None):
    rows, F = gu.shape[0], gu.shape[-1] // 2
    L = lib()
    dgu = torch.empty_like(gu)
    need = L.tkb_swiglu_bwd_workspace(rows, F)
    ws, _ = _ws(need, gu.device)
    check(L.tkb_swiglu_bwd(_p(dh), _p(gu), _p(bg), _p(bu), _p(dgu), _p(dbg), _p(dbu), _p(ws), need, rows, F,
                           dtype_code(gu), _stream()), "tkb_swiglu_bwd")
    return dgu


def qkv_prep_fwd(x, bias, gain, S, Hq, Hkv, D, qknorm=False, rope=True, theta=10000.0, rope_scale=1.0,
                 low=1.0, high=4.0, octx=8192.0):
    rows = x.shape[0]
    out = torch.empty_like(x)
    istd = torch.empty(rows, Hq + Hkv, dtype=torch.float32, device=x.device) if qknorm else None
    check(lib().tkb_qkv_prep_fwd(_p(x), _p(bias), _p(gain), _p(out), _p(istd), rows, S, Hq, Hkv, D, int(qknorm),
                                 int(rope), theta, rope_scale, low, high, octx, dtype_code(x), _stream()),
          "tkb_qkv_prep_fwd")
    return out, istd


def qkv_prep_bwd(dout, x, bias, gain, istd, din, S, Hq, Hkv, D, qknorm=False, rope=True, theta=10000.0,
                 rope_scale=1.0, low=1.0, high=4.0, octx=8192.0, dbias=None, dgain=None):
    rows = x.shape[0]
    L = lib()
    need = L.tkb_qkv_prep_bwd_workspace(rows, Hq, Hkv, D)
    ws, _ = _ws(need, x.device)
    check(L.tkb_qkv_prep_bwd(_p(dout), _p(x), _p(bias), _p(gain), _p(istd), _p(din), _p(dbias), _p(dgain), _p(ws),
                             need, rows, S, Hq, Hkv, D, int(qknorm), int(rope), theta, rope_scale, low, high, octx,
                             dtype_code(x), _stream()), "tkb_qkv_prep_bwd")
    return din


def softmax_fwd(x):
    rows, C = x.shape
    p = torch.empty_like(x)
    check(lib().tkb_softmax_fwd(_p(x), _p(p), rows, C, dtype_code(x), _stream()), "tkb_softmax_fwd")
    return p


def softmax_bwd(p, dp, dx):
    rows, C = p.shape
    check(lib().tkb_softmax_bwd(_p(p), _p(dp), _p(dx), rows, C, dtype_code(p), _stream()), "tkb_softmax_bwd")
    return dx


def softmax_loss(logits, labels, kind=0, gamma=2.0, want_grad=True):
    rows, C = logits.shape
    L = lib()
    dl = torch.empty_like(logits) if want_grad else None
    loss = torch.zeros(1, dtype=torch.float32, device=logits.device)
    corr = torch.zeros(1, dtype=torch.int32, device=logits.device)
    need = L.tkb_softmax_loss_workspace(rows)
    ws, _ = _ws(need, logits.device)
    check(L.tkb_softmax_loss(_p(logits), _p(labels), _p(dl), _p(loss), _p(corr), _p(ws), need, rows, C, kind,
                             gamma, dtype_code(logits), _stream()), "tkb_softmax_loss")
    return loss, dl, corr


class SgdTensor(ctypes.Structure):
    _fields_ = [("master", ctypes.c_void_p), ("vel", ctypes.c_void_p), ("grad", ctypes.c_void_p),
                ("lowp", ctypes.c_void_p), ("n", ctypes.c_longlong), ("apply_wd", ctypes.c_int),
                ("lowp_dtype", ctypes.c_int)]


def sgd_table(entries, device):
    """entries: list of (master, vel, grad, lowp_or_None, apply_wd) -> device table tensor."""
    arr = (SgdTensor * len(entries))()
    for i, (m, v, g, lp, wd) in enumerate(entries):
        arr[i] = SgdTensor(m.data_ptr(), v.data_ptr(), g.data_ptr(), lp.data_ptr() if lp is not None else None,
                           m.numel(), int(wd), dtype_code(lp) if lp is not None else 0)
    host = torch.frombuffer(bytearray(bytes(arr)), dtype=torch.uint8)
    return host.to(device)


def sgd_step(table, n, lr_dev, momentum=0.9, wd=1e-4, seed_dev=None):
    check(lib().tkb_sgd_step(_p(table), n, _p(lr_dev), momentum, wd, _p(seed_dev), _stream()), "tkb_sgd_step")


def gemm(A, B, a_trans=False, b_trans=False, out=None, out_dtype=None, accumulate=False, bias=None):
    """C (+)= op(A) op(B) on the tcgen05 GEMM (tkb_gemm).  A is [M][K] (a_trans:
    [K][M]); B is [K][N] (b_trans: [N][K]); bf16 operands, C bf16 or fp32."""
    M = A.shape[1] if a_trans else A.shape[0]
    K = A.shape[0] if a_trans else A.shape[1]
    N = B.shape[0] if b_trans else B.shape[1]
    if out is None:
        out = torch.empty(M, N, dtype=out_dtype or torch.bfloat16, device=A.device)
    ws, nws = _ws(lib().tkb_gemm_workspace(M, N, K, dtype_code(out)), A.device)
    check(lib().tkb_gemm(_p(A), A.stride(0), int(a_trans), _p(B), B.stride(0), int(b_trans), _p(out), out.stride(0),
                         dtype_code(out), int(accumulate), _p(bias), M, N, K, _p(ws), nws, _stream()), "tkb_gemm")
    return out


def gemm_swiglu(A, B, F, bias_gate=None, bias_up=None):
    """([G|U] bf16 [M][2F], h bf16 [M][F]) with [G|U] = A B and h = SiLU(G + b_g) * (U + b_u)."""
    M, K = A.shape
    gu = torch.empty(M, 2 * F, dtype=torch.bfloat16, device=A.device)
    h = torch.empty(M, F, dtype=torch.bfloat16, device=A.device)
    check(lib().tkb_gemm_swiglu(_p(A), A.stride(0), _p(B), B.stride(0), F, _p(bias_gate), _p(bias_up), _p(gu),
                                gu.stride(0), _p(h), h.stride(0), M, K, _stream()), "tkb_gemm_swiglu")
    return gu, h


def lmhead_ce(X, W, labels, bias=None, want_grad=True):
    """(loss, d logits or None, correct) of softmax cross-entropy over
    logits = X W + bias, without storing the logits (tkb_lmhead_ce)."""
    rows, d = X.shape
    V = W.shape[1]
    loss = torch.zeros(1, dtype=torch.float32, device=X.device)
    corr = torch.zeros(1, dtype=torch.int32, device=X.device)
    dl = torch.empty(rows, V, dtype=torch.bfloat16, device=X.device) if want_grad else None
    ws, nws = _ws(lib().tkb_lmhead_ce_workspace(rows, V), X.device)
    check(lib().tkb_lmhead_ce(_p(X), X.stride(0), _p(W), W.stride(0), _p(bias), _p(labels), _p(dl),
                              dl.stride(0) if dl is not None else 0, _p(loss), _p(corr), _p(ws), nws, rows, d, V,
                              _stream()), "tkb_lmhead_ce")
    return loss, dl, corr


class _KVCacheStruct(ctypes.Structure):
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("pos", ctypes.c_void_p),
                ("weight", ctypes.c_void_p), ("block_table", ctypes.c_void_p), ("seq_lens", ctypes.c_void_p),
                ("page_stride", ctypes.c_longlong), ("n_pages", ctypes.c_int), ("page_size", ctypes.c_int),
                ("max_pages", ctypes.c_int), ("B", ctypes.c_int), ("Hkv", ctypes.c_int), ("D", ctypes.c_int),
                ("dtype", ctypes.c_int)]


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _expect(t, name, shape, dtype):
    if t is not None and (t.shape != shape or t.dtype != dtype or not t.is_contiguous()):
        raise TkbError(f"{name}: expected a contiguous {dtype} tensor of shape {tuple(shape)}, "
                       f"got {t.dtype} {tuple(t.shape)}")


def _vec(t, name, n, dtype):
    """t, if given, holds n contiguous values of dtype."""
    if t is not None and (t.numel() != n or t.dtype != dtype or not t.is_contiguous()):
        raise TkbError(f"{name}: expected {n} contiguous {dtype}, got {t.dtype} {tuple(t.shape)}")


def _row_stride(t, width):
    """Elements from row to row of [rows, width]; a single row's stride means nothing."""
    return t.stride(0) if t.shape[0] > 1 else width


def _launch_stream(who, first, *others):
    """The current stream as an integer (0.2 us; the Stream object of _stream costs 3.4), once all tensors given are
    found on the current CUDA device: a kernel would take any other address for its own memory."""
    dev = first.get_device()
    if dev < 0 or dev != torch._C._cuda_getDevice():
        raise TkbError(f"{who}: expected tensors on the current CUDA device, got one on {first.device}")
    for t in others:
        if t is not None and t.get_device() != dev:
            raise TkbError(f"{who}: expected all tensors on {first.device}, got one on {t.device}")
    return torch._C._cuda_getCurrentRawStream(dev)


class KVCache:
    """One attention layer's paged key-value cache (tkb_kv_cache): tensors
    k, v [n_pages, Hkv, page_size, D] (any page stride, the rest contiguous),
    block_table [B, max_pages] and seq_lens [B] int32, and, for the eviction,
    pos (int32) and weight (fp32) [n_pages, Hkv, page_size]."""

    def __init__(self, k, v, block_table, seq_lens, pos=None, weight=None):
        n_pages, Hkv, page, D = k.shape
        B, max_pages = block_table.shape
        for t, name in ((k, "k"), (v, "v")):
            if tuple(t.shape) != (n_pages, Hkv, page, D) or t.dtype != k.dtype or \
                    t.stride()[2:] != (D, 1) or (Hkv > 1 and t.stride(1) != page * D) or \
                    (n_pages > 1 and t.stride(0) != k.stride(0)):
                raise TkbError(f"{name}: expected {k.dtype} [n_pages, Hkv, page_size, D], contiguous within a page, "
                               "k and v with the same page stride")
        _expect(block_table, "block_table", (B, max_pages), torch.int32)
        _expect(seq_lens, "seq_lens", (B,), torch.int32)
        _expect(pos, "pos", (n_pages, Hkv, page), torch.int32)
        _expect(weight, "weight", (n_pages, Hkv, page), torch.float32)
        for t in (v, block_table, seq_lens, pos, weight):
            if t is not None and t.device != k.device:
                raise TkbError(f"KVCache: expected all tensors on {k.device}, got one on {t.device}")
        self.k, self.v, self.block_table, self.seq_lens, self.pos, self.weight = k, v, block_table, seq_lens, pos, weight
        self.B, self.Hkv, self.D, self.page_size, self.max_pages = B, Hkv, D, page, max_pages
        # a single page has no stride of its own
        stride = k.stride(0) if n_pages > 1 else Hkv * page * D
        self.struct = _KVCacheStruct(k.data_ptr(), v.data_ptr(), pos.data_ptr() if pos is not None else None,
                                     weight.data_ptr() if weight is not None else None, block_table.data_ptr(),
                                     seq_lens.data_ptr(), stride, n_pages, page, max_pages, B, Hkv, D, dtype_code(k))
        self.ref = ctypes.addressof(self.struct)

    @property
    def capacity(self):
        """Tokens a sequence's table has room for."""
        return self.max_pages * self.page_size


def kv_lens(seq_lens, limit=None, seen=None, add=0, row_start=None):
    """seq_lens = min(seq_lens + n, limit) and seen += n, on the device (n = add, or row_start's differences).
    No limit before rows are appended (kv_append leaves out those past the capacity); the budget after an eviction."""
    B = seq_lens.numel()
    _vec(seq_lens, "seq_lens", B, torch.int32)
    _vec(seen, "seen", B, torch.int32)
    _vec(row_start, "row_start", B + 1, torch.int32)
    stream = _launch_stream("kv_lens", seq_lens, seen, row_start)
    check(lib().tkb_kv_lens(seq_lens.data_ptr(), _ptr(seen), _ptr(row_start), int(add),
                            0x7FFFFFFF if limit is None else int(limit), B, stream),
          "tkb_kv_lens")


def kv_append(cache, qkv, Hq, seen=None, row_start=None, bias=None, qk_gain=None, qknorm=False, rope=True,
              theta=10000.0, rope_scale=1.0, low=1.0, high=4.0, octx=8192.0, full=False, out=None):
    """Packed rows qkv [rows, (Hq+2Hkv)*D] enter the cache (tkb_kv_append); returns the prepared query columns
    [rows, Hq*D], or the whole prepared rows with `full`.  seq_lens and seen already count the new rows."""
    if qkv.dtype != cache.k.dtype:
        raise TkbError(f"kv_append: rows are {qkv.dtype}, the cache is {cache.k.dtype}")
    rows = qkv.shape[0]
    C = (Hq + 2 * cache.Hkv) * cache.D
    width = C if full else Hq * cache.D
    if qkv.shape != (rows, C) or qkv.stride(1) != 1:
        raise TkbError(f"kv_append: qkv is {tuple(qkv.shape)}, not rows of {C} contiguous columns")
    _vec(seen, "seen", cache.B, torch.int32)
    _vec(row_start, "row_start", cache.B + 1, torch.int32)
    _vec(bias, "bias", C, torch.float32)
    _vec(qk_gain, "qk_gain", (Hq + cache.Hkv) * cache.D, torch.float32)
    if out is None:
        out = torch.empty(rows, width, dtype=qkv.dtype, device=qkv.device)
    elif out.shape != (rows, width) or out.dtype != qkv.dtype or out.stride(1) != 1:
        raise TkbError(f"kv_append: out is {out.dtype} {tuple(out.shape)}, not {qkv.dtype} {(rows, width)}")
    stream = _launch_stream("kv_append", cache.k, qkv, bias, qk_gain, out, row_start, seen)
    check(lib().tkb_kv_append(cache.ref, _ptr(qkv), _row_stride(qkv, C), _ptr(bias), _ptr(qk_gain), _ptr(out),
                              _row_stride(out, width), int(full), _ptr(row_start), _ptr(seen), rows, Hq, int(qknorm),
                              int(rope), theta, rope_scale, low, high, octx, stream), "tkb_kv_append")
    return out


def paged_attn_workspace(cache, Hq, accumulate=False):
    """Zeroed workspace of paged_attn_decode; one per stream that calls it, the largest of its caches' serving all."""
    n = lib().tkb_paged_attn_decode_workspace(cache.ref, Hq, int(accumulate))
    if n == 0:
        check(-1, "tkb_paged_attn_decode_workspace")
    return torch.zeros(n, dtype=torch.uint8, device=cache.k.device)


def paged_attn_decode(cache, q, Hq, scale=None, accumulate=False, out=None, lse=None, workspace=None):
    """Attention of one token per sequence over its cache: q [B, Hq*D] -> (out [B, Hq*D], lse [B, Hq] fp32)."""
    if q.dtype != cache.k.dtype:
        raise TkbError(f"paged_attn_decode: q is {q.dtype}, the cache is {cache.k.dtype}")
    if q.shape != (cache.B, Hq * cache.D):
        raise TkbError(f"paged_attn_decode: q is {tuple(q.shape)}, not {(cache.B, Hq * cache.D)}")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif out.shape != q.shape or out.dtype != q.dtype:
        raise TkbError(f"paged_attn_decode: out is {out.dtype} {tuple(out.shape)}, not as q")
    if q.stride(1) != 1 or out.stride(1) != 1:
        raise TkbError("paged_attn_decode: columns of q and out must be contiguous")
    if lse is None:
        lse = torch.empty(cache.B, Hq, dtype=torch.float32, device=q.device)
    else:
        _vec(lse, "lse", cache.B * Hq, torch.float32)
    if workspace is None:
        workspace = paged_attn_workspace(cache, Hq, accumulate)
    stream = _launch_stream("paged_attn_decode", cache.k, q, out, lse, workspace)
    width = Hq * cache.D
    check(lib().tkb_paged_attn_decode(cache.ref, _ptr(q), _row_stride(q, width), _ptr(out), _row_stride(out, width),
                                      _ptr(lse), Hq, cache.D ** -0.5 if scale is None else scale, int(accumulate),
                                      _ptr(workspace), workspace.numel(), stream), "tkb_paged_attn_decode")
    return out, lse


def kv_evict_workspace(cache):
    n = lib().tkb_kv_evict_workspace(cache.ref)
    if n == 0:
        check(-1, "tkb_kv_evict_workspace")
    return torch.empty(n, dtype=torch.uint8, device=cache.k.device)


def kv_evict(cache, budget, seen, recent=0, sinks=0, workspace=None):
    """Keep `budget` tokens of every (sequence, kv head) that holds more, by accumulated weight (tkb_kv_evict);
    kv_lens(cache.seq_lens, budget) after the last layer."""
    _vec(seen, "seen", cache.B, torch.int32)
    if workspace is None:
        workspace = kv_evict_workspace(cache)
    stream = _launch_stream("kv_evict", cache.k, seen, workspace)
    check(lib().tkb_kv_evict(cache.ref, _ptr(seen), int(budget), int(recent), int(sinks), _ptr(workspace),
                             workspace.numel(), stream), "tkb_kv_evict")


def sample_logits(logits, u, temperature=None, top_k=None, top_p=None, min_p=None):
    """(token int32, logprob fp32, kept int32) per row of logits [rows, V] from uniform numbers u [rows]
    (tkb_sample_logits); the parameters are per-row tensors (top_k int32, the others fp32) or None."""
    rows, V = logits.shape
    if V > 1 and logits.stride(1) != 1:
        raise TkbError("sample_logits: a row's logits must be contiguous")
    for t, name, dt in ((u, "u", torch.float32), (temperature, "temperature", torch.float32),
                        (top_k, "top_k", torch.int32), (top_p, "top_p", torch.float32), (min_p, "min_p", torch.float32)):
        _expect(t, name, (rows,), dt)
    stream = _launch_stream("sample_logits", logits, u, temperature, top_k, top_p, min_p)
    logprob = torch.empty_like(u)
    token = torch.empty_like(u, dtype=torch.int32)
    kept = torch.empty_like(token)
    check(lib().tkb_sample_logits(_ptr(logits), _row_stride(logits, V), _ptr(u), _ptr(temperature),
                                  _ptr(top_k), _ptr(top_p), _ptr(min_p), _ptr(token), _ptr(logprob), _ptr(kept), rows, V,
                                  dtype_code(logits), stream), "tkb_sample_logits")
    return token, logprob, kept
