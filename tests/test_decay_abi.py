"""CPU checks of the entry points of include/based_la_decay.h: exported, and bad arguments refused on the
host before any launch (no GPU needed)."""

import ctypes
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "based_la_decay.h")
P = ctypes.c_void_p(64)        # non-null, aligned, never read
ODD = ctypes.c_void_p(66)
S3 = ctypes.c_longlong * 3


def _lib():
    from kernels import _lib
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("libbased_la.so not built")
    return _lib.lib()


def test_exports():
    lib = _lib()
    names = re.findall(r"^\s*(?:int|size_t)\s+(la_\w+)\s*\(", open(HEADER).read(), re.M)
    assert sorted(names) == ["la_decay_bwd", "la_decay_fwd", "la_decay_step", "la_decay_workspace_bytes"]
    assert all(hasattr(lib, n) for n in names)


def test_signatures_match_the_headers():
    """The ctypes signature of every entry point: the declaration's arguments, kind by kind."""
    from kernels import _lib
    kinds = {ctypes.c_void_p: "pointer", ctypes.c_float: "float", ctypes.c_size_t: "size", ctypes.c_int: "int",
             ctypes.c_longlong: "long"}
    seen = set()
    for name in ("based_la.h", "based_la_ext.h", "based_la_decay.h", "based_la_cache.h"):
        text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", name)).read(), flags=re.S)
        for fn, args in re.findall(r"(la_\w+)\s*\(([^)]*)\)\s*;", text):
            want = ["pointer" if "*" in a else "float" if a.startswith("float") else "size" if a.startswith("size_t") else
                    "long" if a.startswith("long long") else "int" for a in (x.strip() for x in args.split(",")) if a != "void"]
            assert [kinds[a] for a in _lib._SIGNATURES[fn][1]] == want, fn
            seen.add(fn)
    assert seen == set(_lib._SIGNATURES)


def test_workspace_sizes():
    lib = _lib()
    assert lib.la_decay_workspace_bytes(1, 1, 64, 64, 64, 0) == 0
    assert 0 < lib.la_decay_workspace_bytes(1, 4, 8192, 64, 64, 0) < lib.la_decay_workspace_bytes(1, 4, 8192, 64, 64, 1)
    for bad in ((0, 1, 64, 64, 64), (1, 1, 0, 64, 64), (1, 1, 8192, 129, 64), (1, 1, 8192, 64, 0), (1, -1, 8192, 64, 64)):
        assert lib.la_decay_workspace_bytes(*bad, 0) == 0


FWD = dict(q=P, k=P, v=P, dt=1, out=P, odt=1, B=1, H=2, N=8, d=16, dv=64, qs=None, ks=None, vs=None, g=P, lens=None,
           scale=0.25, si=None, so=None, ws=None, wsb=0)
BWD = dict(q=P, k=P, v=P, do=P, dt=1, dq=P, dk=P, dvo=P, B=1, H=2, N=8, d=16, dv=64, qs=None, ks=None, vs=None, dos=None,
           g=P, lens=None, scale=0.25, si=None, dso=None, dsi=None, fws=None, ws=None, wsb=0)
STEP = dict(q=P, k=P, v=P, dt=1, g=P, state=P, out=P, odt=1, B=1, H=2, d=16, dv=64, scale=0.25)
FAR = ctypes.c_void_p(1 << 20)

COMMON = [(dict(q=None), -1), (dict(k=None), -1), (dict(v=None), -1), (dict(g=None), -1), (dict(B=-1), -2), (dict(d=0), -2),
          (dict(dt=3), -3), (dict(scale=0.0), -4), (dict(scale=1e-40), -4), (dict(scale=float("inf")), -4), (dict(d=129), -5), (dict(dv=129), -5),
          (dict(q=ctypes.c_void_p(65)), -8), (dict(B=1 << 16, H=33), -2)]
SEQ = COMMON + [(dict(N=-1), -2), (dict(N=(1 << 30) + 1), -2), (dict(qs=S3(0, 0, -1)), -2), (dict(si=ODD), -8), (dict(lens=ODD), -8),
                (dict(N=100000), -6), (dict(N=100000, ws=ODD, wsb=1 << 40), -8)]


@pytest.mark.parametrize("kw,code", SEQ + [(dict(out=None), -1), (dict(odt=5), -3), (dict(out=ODD), -8),
                                           (dict(si=P, so=P), -9), (dict(si=P, so=ctypes.c_void_p(128)), -9)])
def test_forward_refusals(kw, code):
    assert _lib().la_decay_fwd(*{**FWD, **kw}.values(), None) == code


@pytest.mark.parametrize("kw,code", SEQ + [(dict(do=None), -1), (dict(dq=None), -1), (dict(dk=None), -1), (dict(dvo=None), -1),
                                           (dict(dk=ODD), -8), (dict(dso=FAR, dsi=FAR), -9),
                                           (dict(N=100000, fws=ODD, ws=P, wsb=1 << 40), -8),
                                           (dict(N=100000, fws=P, ws=P, wsb=1 << 40), -9)])
def test_backward_refusals(kw, code):
    assert _lib().la_decay_bwd(*{**BWD, **kw}.values(), None) == code


@pytest.mark.parametrize("kw,code", COMMON + [(dict(state=None), -1), (dict(out=None), -1), (dict(state=ODD), -8), (dict(odt=9), -3)])
def test_step_refusals(kw, code):
    assert _lib().la_decay_step(*{**STEP, **kw}.values(), None) == code


def test_nothing_to_do():
    lib = _lib()
    assert lib.la_decay_fwd(*{**FWD, "N": 0, "q": None}.values(), None) == 0
    assert lib.la_decay_bwd(*{**BWD, "B": 0}.values(), None) == 0
    assert lib.la_decay_step(*{**STEP, "H": 0}.values(), None) == 0


def test_wrapper_refuses_cpu_tensors():
    import torch

    import kernels
    x = torch.zeros(1, 2, 4, 16)
    with pytest.raises(RuntimeError):
        kernels.decay_linear_attn(x, x, x, torch.zeros(2))
    with pytest.raises(RuntimeError):
        kernels.decay_decode_step(x[:, :, 0], x[:, :, 0], x[:, :, 0], torch.zeros(2), torch.zeros(1, 2, 16, 16))
