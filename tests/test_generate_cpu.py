"""Refusals of the generation entry points: bad arguments are turned down
with a message before any CUDA call."""
import ctypes

import pytest

import tokamak_b200
from tokamak_b200.ops import _KVCacheStruct

vp = ctypes.c_void_p


def cache(**over):
    f = dict(k=256, v=256, pos=256, weight=256, block_table=256, seq_lens=256, page_stride=2 * 16 * 64, n_pages=8,
             page_size=16, max_pages=4, B=2, Hkv=2, D=64, dtype=1)
    f.update(over)
    return _KVCacheStruct(*[f[n] for n, _ in _KVCacheStruct._fields_])


def decode(c, Hq=4, q=256, out=256, stride=256, acc=0, ws=256, n=1 << 30):
    L = tokamak_b200.lib()
    return L.tkb_paged_attn_decode(ctypes.byref(c) if c else None, vp(q), stride, vp(out), stride, None, Hq, 0.1, acc,
                                   vp(ws), n, None)


def append(c, rows=2, Hq=4, qkv=256, stride=8 * 64, out=256, out_stride=8 * 64, full=1, start=None, theta=1e4):
    L = tokamak_b200.lib()
    return L.tkb_kv_append(ctypes.byref(c), vp(qkv), stride, None, None, vp(out), out_stride, full, start, None, rows,
                           Hq, 0, 1, theta, 1.0, 1.0, 4.0, 8192.0, None)


def evict(c, budget=16, recent=4, sinks=4, seen=256, ws=256, n=1 << 30):
    return tokamak_b200.lib().tkb_kv_evict(ctypes.byref(c), vp(seen), budget, recent, sinks, vp(ws), n, None)


def message():
    return tokamak_b200.lib().tkb_last_error().decode()


@pytest.mark.parametrize("over,code", [
    (dict(k=0), -1), (dict(seq_lens=0), -1), (dict(block_table=0), -1), (dict(k=264), -1), (dict(dtype=7), -1),
    (dict(B=0), -1), (dict(B=5000), -3), (dict(D=96), -3), (dict(page_size=24), -1), (dict(page_size=2048), -1),
    (dict(page_size=0), -1), (dict(page_stride=2 * 16 * 64 - 8), -1), (dict(page_stride=2 * 16 * 64 + 4), -1),
    (dict(max_pages=1 << 28), -1), (dict(n_pages=0), -1), (dict(Hkv=0), -1)])
def test_bad_caches(over, code):
    c = cache(**over)
    assert decode(c) == code and message()
    assert append(c) == code and evict(c) == code
    L = tokamak_b200.lib()
    assert L.tkb_paged_attn_decode_workspace(ctypes.byref(c), 4, 0) == 0
    assert L.tkb_kv_evict_workspace(ctypes.byref(c)) == 0


def test_decode_refusals():
    assert decode(None) == -1
    assert decode(cache(), Hq=3) == -1 and "multiple" in message()
    assert decode(cache(), Hq=0) == -1
    assert decode(cache(), q=0) == -1 and decode(cache(), out=0) == -1
    assert decode(cache(), q=264) == -1 and decode(cache(), stride=128) == -1 and decode(cache(), stride=260) == -1
    assert decode(cache(weight=0), acc=1) == -1 and "weight" in message()
    assert decode(cache(), ws=0) == -4 and decode(cache(), n=8) == -4 and decode(cache(), ws=272) == -4


def test_append_refusals():
    assert append(cache(), rows=3) == -1 and "row_start" in message()
    assert append(cache(), rows=0) == -1 and append(cache(), Hq=0) == -1
    assert append(cache(), qkv=0) == -1 and append(cache(), qkv=264) == -1
    assert append(cache(), stride=8 * 64 - 8) == -1 and append(cache(), stride=8 * 64 + 4) == -1
    assert append(cache(), out_stride=4 * 64) == -1
    assert append(cache(), theta=0.0) == -1


def test_evict_refusals():
    assert evict(cache(pos=0)) == -1 and evict(cache(weight=0)) == -1 and evict(cache(), seen=0) == -1
    assert evict(cache(), budget=0) == -1 and evict(cache(), budget=7) == -1 and evict(cache(), recent=-1) == -1
    assert evict(cache(), ws=0) == -4 and evict(cache(), n=4) == -4


def test_lens_refusals():
    L = tokamak_b200.lib()
    assert L.tkb_kv_lens(None, None, None, 1, 10, 4, None) == -1
    assert L.tkb_kv_lens(vp(256), None, None, 1, 10, 0, None) == -1
    assert L.tkb_kv_lens(vp(256), None, None, -1, 10, 4, None) == -1


def test_sample_refusals():
    L = tokamak_b200.lib()

    def call(logits=256, ld=100, u=256, token=256, rows=2, V=100, dtype=0):
        return L.tkb_sample_logits(vp(logits), ld, vp(u), None, None, None, None, vp(token), None, None, rows, V, dtype,
                                   None)
    assert call(logits=0) == -1 and call(u=0) == -1 and call(token=0) == -1
    assert call(rows=0) == -1 and call(V=0) == -1 and call(ld=99) == -1 and call(dtype=3) == -1
    assert call(V=(1 << 20) + 1, ld=1 << 21) == -3
    assert call(logits=258) == -1


def test_python_checks():
    torch = pytest.importorskip("torch")
    from tokamak_b200 import TkbError, ops
    k = torch.zeros(4, 2, 16, 64)
    table, lens = torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    c = ops.KVCache(k, k.clone(), table, lens)
    assert c.capacity == 32
    with pytest.raises(TkbError):
        ops.KVCache(k, k[:, :, :, :32], table, lens)
    with pytest.raises(TkbError):
        ops.KVCache(k.transpose(1, 2), k.transpose(1, 2), table, lens)
    with pytest.raises(TkbError):
        ops.KVCache(k, k.clone(), table.long(), lens)
    with pytest.raises(TkbError):
        ops.KVCache(k, k.clone(), table, lens[:1])
    with pytest.raises(TkbError):
        ops.paged_attn_decode(c, torch.zeros(3, 4 * 64), 4)
    with pytest.raises(TkbError):
        ops.paged_attn_decode(c, torch.zeros(2, 4 * 64, dtype=torch.bfloat16), 4)
    with pytest.raises(TkbError):
        ops.sample_logits(torch.zeros(2, 8), torch.zeros(3))
    with pytest.raises(TkbError):
        ops.sample_logits(torch.zeros(2, 8), torch.zeros(2), top_k=torch.zeros(2))
    q2 = torch.zeros(2, 4 * 64)
    with pytest.raises(TkbError):
        ops.paged_attn_decode(c, q2, 4, out=torch.zeros(2, 64))
    with pytest.raises(TkbError):
        ops.paged_attn_decode(c, q2, 4, lse=torch.zeros(2, 3))
    rows = torch.zeros(2, 8 * 64)
    for bad in (dict(bias=torch.zeros(7)), dict(qk_gain=torch.zeros(8 * 64)), dict(seen=lens.long()),
                dict(row_start=lens), dict(out=torch.zeros(2, 64))):
        with pytest.raises(TkbError):
            ops.kv_append(c, rows, 4, **bad)
    with pytest.raises(TkbError):
        ops.kv_append(c, rows[:, :64], 4)
    with pytest.raises(TkbError):
        ops.kv_evict(c, 8, lens[:1])
    with pytest.raises(TkbError):
        ops.kv_lens(lens.long(), 4)
    with pytest.raises(TkbError):
        ops.kv_lens(lens, 4, row_start=lens)


def test_tensors_of_the_host_are_refused():
    """Right in shape and type, but on the host: an error here instead of a kernel that reads host addresses."""
    torch = pytest.importorskip("torch")
    from tokamak_b200 import TkbError, ops
    k = torch.zeros(4, 2, 16, 64)
    meta = dict(pos=torch.zeros(4, 2, 16, dtype=torch.int32), weight=torch.zeros(4, 2, 16))
    table, lens = torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    c = ops.KVCache(k, k.clone(), table, lens, **meta)
    calls = [lambda: ops.kv_lens(lens, add=1), lambda: ops.kv_append(c, torch.zeros(2, 8 * 64), 4, seen=lens),
             lambda: ops.paged_attn_decode(c, torch.zeros(2, 4 * 64), 4), lambda: ops.kv_evict(c, 8, lens),
             lambda: ops.sample_logits(torch.zeros(2, 8), torch.zeros(2))]
    for call in calls:
        with pytest.raises(TkbError, match="CUDA device"):
            call()
    with pytest.raises(TkbError, match="expected all tensors on cpu"):
        ops.KVCache(k, k.clone(), table, lens.to("meta"), **meta)


def test_tensors_of_another_device_are_refused(monkeypatch):
    """One tensor on another device than the first, or all on another than the current one."""
    torch = pytest.importorskip("torch")
    from tokamak_b200 import TkbError, ops

    class On:
        def __init__(self, i):
            self.i, self.device = i, f"cuda:{i}" if i >= 0 else "cpu"

        def get_device(self):
            return self.i

    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 1, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda dev: 70 + dev, raising=False)
    assert ops._launch_stream("call", On(1), None, On(1)) == 71
    for tensors in ((On(0), On(0)), (On(1), On(0)), (On(1), None, On(-1)), (On(-1), On(1))):
        with pytest.raises(TkbError, match="call"):
            ops._launch_stream("call", *tensors)


def small_generator(**more):
    """A generator whose tensors stay on the host: for what it refuses before it computes anything."""
    pytest.importorskip("torch")
    import numpy as np
    from tokamak_b200 import configs, generate
    cfg = dict(configs.C1, layers=1)
    embed = more.pop("embed", np.zeros((cfg["vocab"], cfg["d_model"]), np.float32))
    return cfg, generate.Generator(cfg, generate.random_checkpoint(cfg), embed, 2, 64, device="cpu", **more)


def test_generator_refuses_token_ids_outside_the_vocabulary():
    """Before the look-up, which would be an assertion on the device."""
    import numpy as np
    from tokamak_b200 import TkbError
    cfg, gen = small_generator()
    for bad in (cfg["vocab"], -1, 1 << 40):
        with pytest.raises(TkbError, match="token ids"):
            gen.prefill([[1, 2], [3, bad]])
    for shape in ((cfg["vocab"] - 1, cfg["d_model"]), (cfg["vocab"], cfg["d_model"] + 1), (cfg["vocab"] * cfg["d_model"],)):
        with pytest.raises(TkbError, match="embed"):
            small_generator(embed=np.zeros(shape, np.float32))


def test_generator_refuses_a_budget_without_room_at_once():
    """recent + sinks above the budget: known before the first token, not at the first cut."""
    from tokamak_b200 import TkbError
    _, gen = small_generator(budget=8, slack=8, recent=6, sinks=4)
    with pytest.raises(TkbError, match="recent"):
        gen.generate([[1] * 10, [2]], 8)   # 16 tokens are held before the eighth


def test_prompts_of_the_command(tmp_path):
    pytest.importorskip("torch")
    from tokamak_b200 import TkbError, generate
    path = tmp_path / "prompts.txt"
    path.write_text("1 2 3\n\n  7\n")
    assert generate.read_prompts(path) == [[1, 2, 3], [7]]
    for bad in ("1 two\n", "\n"):
        path.write_text(bad)
        with pytest.raises(TkbError):
            generate.read_prompts(path)


def test_generator_takes_an_embedding_with_more_rows_than_the_vocabulary():
    import numpy as np
    from tokamak_b200 import TkbError, configs
    V, d = configs.C1["vocab"], configs.C1["d_model"]
    _, gen = small_generator(embed=np.zeros((V + 8, d), np.float32))
    with pytest.raises(TkbError, match=f"0 to {V + 7}"):
        gen.prefill([[V + 8], [0]])
    with pytest.raises(TkbError, match="CUDA device"):  # the ids pass; the tensors are on the host
        gen.prefill([[V + 7], [0]])
