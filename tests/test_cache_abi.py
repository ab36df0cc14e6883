"""CPU checks of the entry points of include/based_la_cache.h: exported, and bad arguments refused on the
host before any launch (no GPU needed)."""

import ctypes
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "based_la_cache.h")
P = ctypes.c_void_p(64)        # non-null, aligned, never read
ODD = ctypes.c_void_p(67)
S3 = ctypes.c_longlong * 3


def _lib():
    from kernels import _lib
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("libbased_la.so not built")
    return _lib.lib()


def test_exports():
    lib = _lib()
    names = re.findall(r"^\s*(?:int|size_t)\s+(la_\w+)\s*\(", open(HEADER).read(), re.M)
    assert sorted(names) == ["la_sliding_cache_append", "la_sliding_cache_dim", "la_sliding_decode_step",
                             "la_sliding_decode_workspace_bytes"]
    assert all(hasattr(lib, n) for n in names)
    assert [lib.la_sliding_cache_dim(d) for d in (0, 1, 32, 33, 64, 65, 128, 129)] == [0, 32, 32, 64, 64, 128, 128, 0]


APPEND = dict(k=P, v=P, dt=1, kc=P, vc=P, ks=P, vs=P, start=None, lens=None, B=1, HK=2, N=8, d=16, dv=64, blocks=4, kst=None,
              vst=None)
STEP = dict(q=P, k=P, v=P, dt=1, out=P, odt=1, kc=P, vc=P, ks=P, vs=P, lens=P, B=1, H=4, HK=2, d=16, dv=64, blocks=4, window=0,
            scale=0.25, ws=None, wsb=0)
BOTH = [(dict(k=None), -1), (dict(v=None), -1), (dict(kc=None), -1), (dict(vs=None), -1), (dict(B=-1), -2), (dict(d=0), -2),
        (dict(blocks=0), -2), (dict(blocks=(1 << 24) + 1), -2), (dict(dt=2), -3), (dict(d=129), -5), (dict(dv=500), -5),
        (dict(kc=ODD), -8), (dict(vc=ctypes.c_void_p(72)), -8), (dict(ks=ODD), -8), (dict(k=ODD), -8), (dict(lens=ODD), -8),
        (dict(B=70000), -2)]


@pytest.mark.parametrize("kw,code", BOTH + [(dict(N=-1), -2), (dict(N=(1 << 29) + 1), -2), (dict(start=ODD), -8), (dict(kst=S3(0, -1, 0)), -2)])
def test_append_refusals(kw, code):
    assert _lib().la_sliding_cache_append(*{**APPEND, **kw}.values(), None) == code


@pytest.mark.parametrize("kw,code", BOTH + [(dict(q=None), -1), (dict(out=None), -1), (dict(lens=None), -1), (dict(H=5), -2),
                                            (dict(HK=0), -2), (dict(window=-1), -2), (dict(window=194), -2), (dict(B=300, H=60000), -2), (dict(odt=7), -3),
                                            (dict(scale=0.0), -4), (dict(scale=float("nan")), -4),
                                            (dict(blocks=4096), -6), (dict(blocks=4096, ws=ODD, wsb=1 << 40), -8)])
def test_step_refusals(kw, code):
    assert _lib().la_sliding_decode_step(*{**STEP, **kw}.values(), None) == code


def test_nothing_to_do():
    lib = _lib()
    assert lib.la_sliding_cache_append(*{**APPEND, "N": 0, "k": None}.values(), None) == 0
    assert lib.la_sliding_decode_step(*{**STEP, "B": 0, "q": None}.values(), None) == 0
    assert lib.la_sliding_decode_workspace_bytes(0, 4, 2, 16, 64, 4, 0) == 0
    assert lib.la_sliding_decode_workspace_bytes(1, 5, 2, 16, 64, 4096, 0) == 0
    assert lib.la_sliding_decode_workspace_bytes(1, 4, 2, 16, 64, 4096, 0) > 0


def test_wrapper_refuses_cpu_tensors():
    import torch

    import kernels
    cache = kernels.sliding_cache(1, 2, 100, 16, device="cpu")
    assert cache.tokens == 128 and cache.k.shape == (1, 2, 2, 64, 32) and cache.v.shape == (1, 2, 2, 32, 64)
    x = torch.zeros(1, 2, 16)
    with pytest.raises(RuntimeError):
        kernels.sliding_decode_step(x, x, x, cache, torch.ones(1, dtype=torch.int32))
    with pytest.raises(RuntimeError):
        kernels.sliding_cache_append(cache, x.unsqueeze(2), x.unsqueeze(2))
    with pytest.raises(RuntimeError):
        kernels.sliding_cache(1, 2, 100, 129, device="cpu")
