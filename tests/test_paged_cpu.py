"""Refusals of the paged cache's entry points without a GPU: the Python wrappers'
argument checks on CPU tensors, and the C entries' host checks (they return
before any launch)."""
import pytest
import torch

from chessdecoder_b200 import _lib
from chessdecoder_b200 import kernels as K

from paged_reference import e4m3, quantise


def _z(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


I32 = torch.int32
K4 = dict(k=_z(4, 2, 16, 64), v=_z(4, 2, 16, 64), table=_z(3, 2, dtype=I32))


def _attn(**kw):
    a = {**K4, "q": _z(3, 256), "lens": _z(3, dtype=I32), "out": _z(3, 256), "ks": None, "vs": None, **kw}
    K.paged_attn(a["q"], a["k"], a["v"], a["table"], a["lens"], a["out"], k_scale=a["ks"], v_scale=a["vs"],
                 workspace=a.get("workspace"))


@pytest.mark.parametrize("kw,why", [
    (dict(v=_z(4, 2, 8, 64)), "alike"), (dict(k=_z(4, 2, 16, 32), v=_z(4, 2, 16, 32)), "alike"),
    (dict(k=_z(4, 2, 16, 64, dtype=torch.float16), v=_z(4, 2, 16, 64, dtype=torch.float16)), "bfloat16 or"),
    (dict(k=_z(4, 16, 2, 64).transpose(1, 2), v=_z(4, 16, 2, 64).transpose(1, 2)), "contiguous"),
    (dict(ks=_z(4, 2, 16, dtype=torch.uint8), vs=_z(4, 2, 16, dtype=torch.uint8)), "no scales"),
    (dict(k=_z(4, 2, 16, 64, dtype=torch.uint8).view(torch.float8_e4m3fn),
          v=_z(4, 2, 16, 64, dtype=torch.uint8).view(torch.float8_e4m3fn)), "need k_scale"),
    (dict(table=_z(3, 2, dtype=torch.int64)), "table"), (dict(table=_z(2, 3, dtype=I32).t()), "table"),
    (dict(lens=_z(2, dtype=I32)), "lens"), (dict(lens=_z(3, dtype=torch.int64)), "lens"),
    (dict(q=_z(3, 128)), "q must be"), (dict(q=_z(3, 256, dtype=torch.float32)), "q must be"),
    (dict(out=_z(3, 192), q=_z(3, 192)), "multiple of"), (dict(out=_z(3, 100), q=_z(3, 100)), "H \\* 64"),
    (dict(out=_z(3, 64 * 34), q=_z(3, 64 * 34)), "at most 16"),
    (dict(table=_z(3, 99, dtype=I32), workspace=_z(1, dtype=torch.uint8)), "workspace"),
    (dict(), "need CUDA tensors"),
])
def test_attn_refuses(kw, why):
    with pytest.raises(RuntimeError, match=why):
        _attn(**kw)


@pytest.mark.parametrize("kw,why", [
    (dict(qkv=_z(6, 500)), "qkv"), (dict(qkv=_z(5, 512)), "qkv"), (dict(start=_z(2, dtype=I32)), "start"),
    (dict(num_new=_z(4, dtype=I32)), "num_new"), (dict(pos=_z(6, dtype=I32)), "go together"),
    (dict(pos=_z(3, dtype=I32), rope=_z(8, 32, 2, dtype=torch.float32)), "pos"),
    (dict(pos=_z(6, dtype=I32), rope=_z(8, 64, 2, dtype=torch.float32)), "rope"),
    (dict(q_out=_z(6, 200)), "q_out"), (dict(), "need CUDA tensors"),
])
def test_append_refuses(kw, why):
    a = dict(qkv=_z(6, 512), start=_z(3, dtype=I32), num_new=None, pos=None, rope=None, q_out=None)
    a.update(kw)
    with pytest.raises(RuntimeError, match=why):
        K.paged_append(a.pop("qkv"), 3, 2, 4, K4["k"], K4["v"], K4["table"], a.pop("start"), **a)


@pytest.mark.parametrize("ko,vo,why", [
    (_z(3, 2, 9, 32), _z(3, 2, 9, 32), "alike"), (_z(3, 2, 9, 64), _z(3, 2, 8, 64), "alike"),
    (_z(3, 1, 9, 64), _z(3, 1, 9, 64), "alike"), (_z(3, 2, 1, 64).expand(3, 2, 9, 64),) * 2 + ("overlap",),
    (_z(3, 2, 9, 64), _z(3, 2, 9, 64), "need CUDA tensors"),
])
def test_gather_refuses(ko, vo, why):
    with pytest.raises(RuntimeError, match=why):
        K.paged_gather(K4["k"], K4["v"], K4["table"], _z(3, dtype=I32), ko, vo)


def _cache(**kw):
    c = dict(k=4096, v=8192, k_scale=0, v_scale=0, table=64, ldt=200, width=200, num_pages=4, ld_page=2 * 16 * 64,
             ld_scale=0, kv_heads=2, page_size=16, dtype=0, reserved=0)
    return _lib.PAGED_CACHE.pack(*{**c, **kw}.values())


#: refused by the C entries before anything is launched (the addresses are never followed)
BAD_CACHE = [(dict(k=0), -1), (dict(table=0), -1), (dict(dtype=2), -2), (dict(dtype=1), -3),
             (dict(page_size=12), -4), (dict(page_size=0), -4), (dict(kv_heads=0), -4), (dict(num_pages=0), -5),
             (dict(ldt=199), -5), (dict(ld_page=2000), -6), (dict(ld_page=2 * 16 * 64 + 4), -6), (dict(k=4100), -7)]


@pytest.mark.parametrize("kw,rc", BAD_CACHE)
def test_c_entries_refuse_a_bad_cache(kw, rc):
    lib, c = _lib.load(), _cache(**kw)
    assert lib.cdk_paged_attn(64, 128, c, 3, 2, 64, 64, 128, 0.125, 64, 1 << 30, None) == rc
    assert lib.cdk_paged_append(64, 384, 0, None, None, 0, 3, 1, 2, c, 64, None, None, 0, None) == rc
    assert lib.cdk_paged_gather(c, 3, 64, 64, 64, 64, 64, 64, 5, None) == rc


def test_c_entries_refuse_bad_arguments():
    lib, c = _lib.load(), _cache()
    attn = lambda q=64, ldq=128, B=3, H=2, out=64, ldo=128, scale=0.125, ws=64, n=1 << 40: lib.cdk_paged_attn(  # noqa: E731
        q, ldq, c, B, H, 64, out, ldo, scale, ws, n, None)
    assert attn(q=None) == -10 and attn(H=3) == -11 and attn(H=34) == -11 and attn(B=20000) == -11
    assert attn(ws=None) == -12 and attn(ws=72) == -12 and attn(n=0) == -12
    assert attn(ldq=120) == -13 and attn(q=68) == -13 and attn(ldo=132) == -13 and attn(scale=float("nan")) == -14
    assert attn(B=0) == 0
    app = lambda qkv=64, ldq=384, f32=0, pos=None, rope=None, n=0, B=3, S=1, H=2, start=64, qo=None, ldo=0: (  # noqa: E731
        lib.cdk_paged_append(qkv, ldq, f32, pos, rope, n, B, S, H, c, start, None, qo, ldo, None))
    assert app(start=None) == -10 and app(ldq=380) == -11 and app(ldq=388) == -11 and app(qkv=72) == -11
    assert app(rope=64) == -12 and app(rope=64, pos=64) == -12 and app(qo=64, ldo=100) == -13
    assert app(B=1 << 39, S=4) == -14 and app(S=0) == 0
    gat = lambda B=3, sb=64, S=5, ko=64: lib.cdk_paged_gather(c, B, 64, ko, 64, sb, 64, 64, S, None)  # noqa: E731
    assert gat(ko=None) == -10 and gat(sb=60) == -11 and gat(ko=72) == -11 and gat(B=70000) == -12 and gat(S=0) == 0
    assert lib.cdk_paged_attn_workspace(3, 5, 2, 9) == -1 and lib.cdk_paged_attn_workspace(3, 4, 2, -1) == -1
    assert lib.cdk_paged_attn_workspace(3, 4, 2, 5000) > 0 and lib.cdk_paged_attn_workspace(3, 4, 2, 64) == 0


def test_the_tests_own_e4m3_is_torchs():
    x = torch.randn(4096, 64) * 100
    assert torch.equal(e4m3(x.double().clamp(-448, 448)), x.clamp(-448, 448).to(torch.float8_e4m3fn).double())
    v, e = quantise(x)
    top = x.double().abs().amax(-1)
    unit = torch.pow(torch.tensor(2.0, dtype=torch.float64), e.double())
    assert (top <= 448 * unit).all() and (top > 224 * unit).all()
    assert ((v - x).abs() <= (2.0 ** -4 * x.abs()).double().maximum(2.0 ** -10 * unit[:, None])).all()


def test_calls_launch_on_the_tensors_device(monkeypatch):
    """A call on tensors of another device than the current one makes that device
    current around the launch and takes its stream."""
    seen, current = [], [0]

    class Device:
        def __init__(self, i):
            self.i = i

        def __enter__(self):
            self.was, current[0] = current[0], self.i

        def __exit__(self, *a):
            current[0] = self.was

    monkeypatch.setattr(K, "_current_device", lambda: current[0])
    monkeypatch.setattr(K, "_raw_stream", lambda dev: 100 + dev)
    monkeypatch.setattr(torch.cuda, "device", Device)
    fn = lambda *a: seen.append((current[0], a)) or 0  # noqa: E731
    K._call("op", fn, 0, 7)
    K._call("op", fn, 3, 8)
    assert seen == [(0, (7, 100)), (3, (8, 103))] and current[0] == 0
    with pytest.raises(RuntimeError, match="op failed with status -5"):
        K._call("op", lambda *a: -5, 0)


def test_layouts_of_different_devices_are_refused():
    lay = lambda dev: (torch.float32, (3,), (1,), dev)  # noqa: E731
    assert K._on("op", lay(1), None, lay(1)) == 1
    with pytest.raises(RuntimeError, match="different devices"):
        K._on("op", lay(1), lay(0))
    with pytest.raises(RuntimeError, match="need CUDA tensors"):
        K._on("op", lay(-1), lay(-1))
