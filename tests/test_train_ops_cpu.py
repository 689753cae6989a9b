"""CPU: the training operators' refusals and ABI.  The argument checks of the C entry points need no GPU; the Python checks are run on
tensors that claim to be on one."""
import ctypes
import os
import subprocess

import pytest
import torch

from diffbir_amd import native, ops, plan

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


@pytest.fixture()
def no_launch(monkeypatch):
    """Host checks only: tensors pass as GPU tensors and every C entry point records its call."""
    calls = []

    class Lib:
        def __getattr__(self, name):
            def call(*a):
                if not name.endswith("_ws"):
                    calls.append(name)
                return 0
            return call

    monkeypatch.setattr(ops, "_gpu", lambda *ts: None)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda dev: 0, raising=False)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: -1)
    ops._ws_bytes.cache_clear()
    monkeypatch.setattr(native, "_lib", Lib())
    yield calls
    ops._ws_bytes.cache_clear()


def qkv(B=2, Lq=5, Lk=7, H=4, Hkv=2, dt=F16):
    return torch.zeros(B, Lq, H, 64, dtype=dt), torch.zeros(B, Lk, Hkv, 64, dtype=dt), torch.zeros(B, Lk, Hkv, 64, dtype=dt)


def test_needs_gpu_tensors():
    q, k, v = qkv()
    with pytest.raises(native.NativeError):
        ops.attention_fwd(q, k, v, 0.125)
    with pytest.raises(native.NativeError):
        ops.layernorm_fwd(torch.zeros(2, 8), torch.ones(8), torch.zeros(8))
    with pytest.raises(native.NativeError):
        ops.embedding(torch.zeros(2, 3, dtype=torch.int64), torch.zeros(4, 8))


def test_attention_refusals(no_launch):
    q, k, v = qkv()
    bad = [
        (q[..., :32], k, v, {}), (q[0], k, v, {}), (q, k[:, :6], v, {}), (q, k, v[:1], {}), (q, k.to(BF16), v, {}),
        (q.double(), k.double(), v.double(), {}), (q, k, v, dict(q_len=torch.zeros(2))), (q, k, v, dict(kv_len=torch.zeros(3, dtype=torch.int32))),
        (q, k, v, dict(kv_len=torch.zeros(4, dtype=torch.int32)[::2])), (q, k, v, dict(out=torch.zeros(2, 5, 4, 64))),
        (torch.zeros(2, 5, 4, 128, dtype=F16)[..., ::2], k, v, {})]
    for a, b, c, kw in bad:
        with pytest.raises((ValueError, TypeError)):
            ops.attention_fwd(a, b, c, 0.125, **kw)
    o, lse = ops.attention_fwd(q, k, v, 0.125)
    g = torch.zeros_like(q)
    for args, kw in [((g[:, :4], q, k, v, o, lse), {}), ((g, q, k, v, o, lse[:1]), {}), ((g, q, k, v, o, lse.double()), {}),
                     ((g, q, k, v, o, lse), dict(dk=torch.zeros_like(q)))]:
        with pytest.raises((ValueError, TypeError)):
            ops.attention_bwd(*args, 0.125, **kw)
    assert no_launch == ["dbir_attention_fwd"]


def test_layernorm_refusals(no_launch):
    x, one = torch.zeros(4, 8), torch.ones(8)
    for args, kw in [((x.double(), one, one), {}), ((x, one[:4], one), {}), ((x, one.half(), one), {}),
                     ((x, one, one), dict(out=x.half())), ((torch.zeros(8, 4).t(), torch.ones(8), torch.ones(8)), {}),
                     ((torch.zeros(1, 8).expand(4, 8), one, one), dict(out=torch.zeros(1, 8).expand(4, 8)))]:
        with pytest.raises((ValueError, TypeError)):
            ops.layernorm_fwd(*args, **kw)
    _, st = ops.layernorm_fwd(x, one, one)
    dy = torch.zeros(4, 8)
    for args, kw in [((dy.half(), x, one, st), {}), ((dy, x, one, st[:2]), {}), ((dy, x, one, st), dict(dres=x.half())), ((dy[:2], x, one, st), {})]:
        with pytest.raises((ValueError, TypeError)):
            ops.layernorm_bwd(*args, **kw)
    assert no_launch == ["dbir_layernorm_fwd"]


def test_embedding_refusals(no_launch):
    tok, table = torch.zeros(2, 3, dtype=torch.int64), torch.zeros(5, 8)
    for args, kw in [((tok.int(), table), {}), ((tok.t(), table), {}), ((tok, table[0]), {}), ((tok, table), dict(pos=torch.zeros(2, 8))),
                     ((tok, table), dict(pos=torch.zeros(3, 8).half())), ((tok, table), dict(out=torch.zeros(2, 3, 7))), ((tok, table.double()), {}),
                     ((tok, table), dict(out=torch.zeros(2, 3, 8), dtype=F16)), ((tok, table.t()), {})]:
        with pytest.raises((ValueError, TypeError)):
            ops.embedding(*args, **kw)
    dy = torch.zeros(2, 3, 8)
    for args, kw in [((dy[:1], tok, 5), {}), ((dy, tok, 0), {}), ((dy, tok, 5), dict(padding_idx=5)), ((dy, tok, 5), dict(padding_idx=-1)),
                     ((dy, tok, 5), dict(accumulate=True)), ((dy, tok, 5), dict(out=torch.zeros(5, 8).half())), ((dy, tok, 5), dict(out=torch.zeros(4, 8))),
                     ((dy.double(), tok, 5), {}), ((dy, tok, 5), dict(pos_rows=1 << 23)), ((dy, tok, 5), dict(pos_rows=-1)), ((dy, tok, 1 << 31), {})]:
        with pytest.raises((ValueError, TypeError)):
            ops.embedding_bwd(*args, **kw)
    assert no_launch == []


def test_refused_while_a_plan_is_recorded(no_launch, monkeypatch):
    monkeypatch.setattr(plan, "_REC", object())
    q, k, v = qkv()
    for call in (lambda: ops.attention_fwd(q, k, v, 0.125), lambda: ops.layernorm_fwd(torch.zeros(2, 8), torch.ones(8), torch.zeros(8)),
                 lambda: ops.embedding(torch.zeros(1, 2, dtype=torch.int64), torch.zeros(4, 8))):
        with pytest.raises(ValueError, match="recorded"):
            call()


def test_row_stride():
    t = torch.zeros(6, 4, 10)
    assert ops._row_ld(t, "t") == 10 and ops._row_ld(t[:, :, :8], "t") == 10 and ops._row_ld(t[:, 0], "t") == 40 and ops._row_ld(t[:1, 1:2], "t") == 10
    assert ops._row_ld(t[:, 1:2, :3], "t") == 40
    for bad in (t[:, :3], t.transpose(0, 2), t[:, :, ::2], t[0, :1].expand(5, 10)):
        with pytest.raises(ValueError):
            ops._row_ld(bad, "t")


# ---- C entry points: every refusal comes before the first launch --------------------------------------------------------
@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(native.LIB_PATH):
        subprocess.run(["sh", os.path.join(ROOT, "diffbir_amd", "csrc", "build.sh")], check=True)
    return native.lib()


def test_attn_desc_layout_matches_header(tmp_path):
    names = [n for n, _ in native.AttnDesc._fields_]
    prog = tmp_path / "sz.c"
    prog.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "%s"\nint main(){printf("%%zu", sizeof(dbir_attn_desc));%s return 0;}'
                    % (os.path.join(ROOT, "include", "dbir.h"), "".join('printf(" %%zu", offsetof(dbir_attn_desc, %s));' % f for f in names)))
    exe = tmp_path / "sz"
    subprocess.run(["gcc", str(prog), "-o", str(exe)], check=True)
    out = [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    assert out[0] == ctypes.sizeof(native.AttnDesc) and out[1:] == [getattr(native.AttnDesc, n).offset for n in names]


def good_desc():
    s = (64 * 128, 128, 64)
    p = [(i + 1) << 20 for i in range(10)]
    return native.AttnDesc(0, 2, 2, 2, 64, 64, 0, 0.125, *p[:5], None, None, *p[5:], 1 << 30, s, s, s, s, s, s, s, s)


@pytest.mark.parametrize("change", [
    dict(dtype=2), dict(dtype=-1), dict(B=0), dict(H=0), dict(Hkv=0), dict(H=3, Hkv=2), dict(Lq=0), dict(Lk=0), dict(Lk=-1), dict(B=70000),
    dict(scale=0.0), dict(scale=1e-31), dict(scale=-1.0), dict(scale=float("inf")), dict(scale=float("nan")), dict(q=None), dict(k=None), dict(v=None), dict(out=None),
    dict(lse=None), dict(q=(1 << 20) + 2), dict(q_stride=(0, 60, 64)), dict(k_stride=(0, 32, 64)), dict(v_stride=(0, 1 << 23, 64)),
    dict(out_stride=(0, 64, 4)), dict(q_stride=(-64, 64, 64)), dict(k_stride=(8192, 128, 4)), dict(dq_stride=(0, 128, 64)), dict(dv_stride=(8192, 128, 0)), dict(dq_stride=(8192, 128, 8)), dict(dk_stride=(56, 128, 64)), dict(dq_stride=(8192, 64, 64)), dict(dk_stride=(64, 128, 64)), dict(dv_stride=(8128, 128, 64)), dict(dq_stride=(4096, 128, 4096)), dict(dq=1 << 20), dict(dk=6 << 20),
    dict(dv=2 << 20), dict(dq=8 << 20, dk=8 << 20), dict(dv=7 << 20), dict(dout=None), dict(dq=None), dict(dk=(1 << 20) + 8), dict(dv_stride=(0, 0, 64)),
    dict(ws=None, Lk=129, B=1), dict(ws_bytes=16, Lk=129, B=1), dict(ws=(1 << 20) + 4, Lk=129, B=1)])
def test_attention_descriptor_refusals(lib, change):
    d = good_desc()
    for n, v in change.items():
        setattr(d, n, (ctypes.c_longlong * 3)(*v) if isinstance(v, tuple) else v)
    assert lib.dbir_attention_bwd(ctypes.byref(d), None) == 1
    assert b"dbir_attention_bwd" in lib.dbir_last_error()
    if not set(change) & {"dout", "dq", "dk", "dv", "dv_stride", "dq_stride", "dk_stride", "ws", "ws_bytes"}:
        assert lib.dbir_attention_fwd(ctypes.byref(d), None) == 1
    assert lib.dbir_attention_fwd(None, None) == 1


def test_attention_forward_refuses_its_input_as_output(lib):
    for name, v in (("out", 1 << 20), ("out", 2 << 20), ("out", 3 << 20), ("out_stride", (8192, 0, 64)), ("out_stride", (0, 128, 64))):
        d = good_desc()
        setattr(d, name, (ctypes.c_longlong * 3)(*v) if isinstance(v, tuple) else v)
        assert lib.dbir_attention_fwd(ctypes.byref(d), None) == 1


def test_packed_descriptor_is_the_struct():
    d = good_desc()
    vals = [getattr(d, n) for n, _ in native.AttnDesc._fields_]
    flat = [x for v in vals for x in (list(v) if hasattr(v, "__len__") else [0 if v is None else v])]
    assert ops._ATTN_PACK(*flat) == bytes(d)


def test_norm_and_embedding_refusals(lib):
    p, r, t, big = 1 << 20, 2 << 20, 3 << 20, 1 << 30
    fwd = [0, p, 8, r, 8, p, p, p, 4, 8, 1e-5, None]
    for i, v in [(0, 3), (0, -1), (1, None), (2, 7), (3, None), (3, p), (4, 7), (5, None), (7, None), (8, 0), (9, 0), (8, (1 << 30) + 1), (10, -1.0), (10, float("nan"))]:
        a = list(fwd)
        a[i] = v
        assert lib.dbir_layernorm_fwd(*a) == 1, (i, v)
    bwd = [0, p, 8, r, 8, None, 0, t, 8, p, p, p, p, 4000, 8, p, big, None]
    for i, v in [(0, 3), (1, None), (2, 7), (4, 7), (5, p), (7, p), (7, r), (8, 7), (9, None), (10, None), (11, None), (12, None), (13, 0), (14, 0), (15, None), (16, 8)]:
        a = list(bwd)
        a[i] = v
        assert lib.dbir_layernorm_bwd(*a) == 1, (i, v)
    a = list(fwd)
    a[2] = a[4] = a[9] = (1 << 28) + 1   # columns
    assert lib.dbir_layernorm_fwd(*a) == 1
    n = ctypes.c_longlong()
    assert lib.dbir_layernorm_bwd_ws(4, (1 << 28) + 1, ctypes.byref(n)) == 1 and lib.dbir_layernorm_bwd_ws(4, 1 << 28, ctypes.byref(n)) == 0
    emb = [2, p, 8, p, None, 0, 2, r, 8, 1.0, 6, 3, 8, 5, None]
    for i, v in [(0, 3), (1, None), (2, 7), (3, None), (4, p), (6, 3), (7, None), (7, p), (8, 7), (10, 0), (11, 0), (12, 0), (13, 0), (10, 1 << 30)]:
        a = list(emb)
        a[i] = v
        assert lib.dbir_embedding_fwd(*a) == 1, (i, v)
    eb = [2, p, 8, p, r, 8, None, 1.0, 6, 3, 8, 5, 0, -1, 0, p, big, None]
    for i, v in [(0, 3), (1, None), (2, 7), (3, None), (4, None), (4, p), (5, 7), (8, 0), (8, 7), (9, 0), (10, 0), (11, 0), (12, 3), (12, 2), (15, None), (16, 8), (15, p + 4)]:
        a = list(eb)
        a[i] = v
        assert lib.dbir_embedding_bwd(*a) == 1, (i, v)
    a = list(eb)
    a[6], a[12] = p, 1 << 23
    assert lib.dbir_embedding_bwd(*a) == 1


def test_training_operators_are_not_recordable(lib):
    for n in ("dbir_attention_fwd", "dbir_attention_bwd", "dbir_layernorm_fwd", "dbir_layernorm_bwd", "dbir_embedding_fwd", "dbir_embedding_bwd"):
        assert lib.dbir_plan_fn_index(n.encode()) == -1
