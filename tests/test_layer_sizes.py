"""Sizes whose products do not fit 64 bits are refused like others that are too large."""
import ctypes

import pytest


@pytest.fixture(scope="module")
def lib():
    from crystalformer_b200 import build
    build.build()
    from crystalformer_b200 import _lib
    return _lib


def test_norms_of_too_many_rows_and_pairs(lib):
    good = dict(type=0, interleaved=0, N=4, Hq=4, Hk=2, D=16, P=8, C=3, wave_heads=1, q=4096, q_row=64, q_head=16, k=4096, k_row=32, k_head=16,
                wq=None, wq_head=0, wk=None, wk_head=0, pos=4096, waves=4096, eps=1e-6)
    for change, code in ((dict(N=2 ** 62, Hq=2, Hk=2), -4), (dict(N=2 ** 63 - 1), -4), (dict(Hk=2 ** 62), -4), (dict(P=2 ** 62), -1), (dict(P=2 ** 63 - 1), -1),
                         (dict(wave_heads=-1), -1), (dict(C=2 ** 62), -2)):
        args = lib.QkNorm(**dict(good, **change))
        for name, rest in (("cf_qk_norm_fwd", (4096, 4096, None)), ("cf_qk_norm_bwd", (4096, 4096, 4096, 4096, None, None, 4096, None))):
            with pytest.raises(lib.CrystalformerB200Error) as e:
                lib.call(name, ctypes.byref(args), *rest)
            assert e.value.code == code, change
        assert lib.load().cf_qk_norm_bwd_workspace_bytes(ctypes.byref(args)) == 0


def test_other_operators_of_too_many_rows(lib):
    for N, V, D in ((2 ** 63 - 1, 4, 8), (4, 2 ** 63 - 1, 8), (4, 4, 2 ** 63 - 1), (2 ** 30, 4, 65536)):
        for name, args in (("cf_embed_fwd", (4096, 8, 1, 0, 4096, N, V, D, 1.0, 4096, None)), ("cf_embed_bwd", (4096, 8, 0, 4096, N, V, D, 1.0, 4096, 0, 4096, None))):
            with pytest.raises(lib.CrystalformerB200Error) as e:
                lib.call(name, *args)
            assert e.value.code == -4
    good = dict(type=1, activation=0, N=4, D=16, F=24, x=4096, ldx=16, w_gate=4096, w_up=4096, w_down=4096, b_gate=None, b_up=None, b_down=None)
    for change in (dict(N=2 ** 63 - 1), dict(D=2 ** 63 - 1), dict(F=2 ** 63 - 1)):
        with pytest.raises(lib.CrystalformerB200Error) as e:
            lib.call("cf_gated_ffn_fwd", ctypes.byref(lib.GatedFFN(**dict(good, **change))), 4096, 4096, None)
        assert e.value.code == -4
