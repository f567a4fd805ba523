"""Operators of a layer beside the attention: what is refused before the device is touched, and layouts that the host decides."""
import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from crystalformer_b200 import build
    build.build()
    from crystalformer_b200 import _lib
    return _lib


def test_cpu_tensors_are_refused():
    from crystalformer_b200.embedding import embed_species
    from crystalformer_b200.feedforward import gated_feed_forward
    from crystalformer_b200.qk_norm import normalize_rotate
    z = torch.zeros
    for call in (lambda: embed_species(z(3, dtype=torch.int64), z(4, 8)), lambda: normalize_rotate(z(3, 2, 4), z(3, 2, 4)),
                 lambda: gated_feed_forward(z(3, 4), z(5, 4), z(5, 4), z(4, 5))):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


def test_positions_and_waves_that_ask_for_gradients_are_refused():
    """They would get none, and nothing would say so."""
    from crystalformer_b200.qk_norm import normalize_rotate
    q, k, pos, waves = torch.zeros(3, 2, 4), torch.zeros(3, 2, 4), torch.zeros(3, 1), torch.zeros(1, 2, 1)
    for args in ((pos.clone().requires_grad_(), waves), (pos, waves.clone().requires_grad_())):
        with pytest.raises(ValueError, match="detach"):
            normalize_rotate(q, k, None, None, *args)
        with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU path"):
            normalize_rotate(q, k, None, None, *args)


def code_of(lib, name, *args):
    with pytest.raises(lib.CrystalformerB200Error) as e:
        lib.call(name, *args)
    return e.value.code


def test_embedding_arguments(lib):
    p = 4096  # (an address that a refused call does not look at)
    assert code_of(lib, "cf_embed_fwd", p, 8, 1, 3, p, 4, 4, 8, 1.0, p, None) == -2
    assert code_of(lib, "cf_embed_fwd", p, 8, 1, 0, p, -1, 4, 8, 1.0, p, None) == -1
    assert code_of(lib, "cf_embed_fwd", p, 8, 1, 0, p, 4, 0, 8, 1.0, p, None) == -1
    assert code_of(lib, "cf_embed_fwd", None, 8, 1, 0, p, 4, 4, 8, 1.0, p, None) == -1
    assert code_of(lib, "cf_embed_fwd", p, -8, 1, 0, p, 4, 4, 8, 1.0, p, None) == -1
    assert code_of(lib, "cf_embed_fwd", p, 8, 1, 0, p, 2 ** 31, 4, 8, 1.0, p, None) == -4
    assert code_of(lib, "cf_embed_fwd", p, 8, 1, 0, p, 4, 4, 65537, 1.0, p, None) == -4
    assert code_of(lib, "cf_embed_bwd", p, 8, 0, p, 4, 4, 8, 1.0, None, 0, p, None) == -1
    assert code_of(lib, "cf_embed_bwd", p, 8, 5, p, 4, 4, 8, 1.0, p, 0, p, None) == -2
    lib.call("cf_embed_fwd", None, 8, 1, 0, None, 0, 4, 8, 1.0, None, None)  # no rows: nothing to do
    assert lib.load().cf_embed_bwd_workspace_bytes(1000, 128) >= 32 * 2 * 128 * 4


def test_norm_arguments(lib):
    good = dict(type=0, interleaved=0, N=4, Hq=4, Hk=2, D=16, P=8, C=3, wave_heads=1, q=4096, q_row=64, q_head=16, k=4096, k_row=32, k_head=16,
                wq=None, wq_head=0, wk=None, wk_head=0, pos=4096, waves=4096, eps=1e-6)
    for change, code in ((dict(type=7), -2), (dict(Hq=3), -1), (dict(P=9), -1), (dict(D=513, P=0), -4), (dict(C=4), -2), (dict(wave_heads=3), -1),
                         (dict(q=None), -1), (dict(waves=None), -1), (dict(q_row=-1), -1), (dict(wq_head=3), -1), (dict(N=-1), -1), (dict(N=2 ** 40), -4)):
        args = lib.QkNorm(**dict(good, **change))
        assert code_of(lib, "cf_qk_norm_fwd", ctypes.byref(args), 4096, 4096, None) == code, change
        assert lib.load().cf_qk_norm_bwd_workspace_bytes(ctypes.byref(args)) == 0
    assert code_of(lib, "cf_qk_norm_fwd", ctypes.byref(lib.QkNorm(**good)), None, 4096, None) == -1
    assert code_of(lib, "cf_qk_norm_bwd", ctypes.byref(lib.QkNorm(**good)), 4096, 4096, 4096, 4096, 4096, None, 4096, None) == -1  # no such weights
    assert code_of(lib, "cf_qk_norm_fwd", None, 4096, 4096, None) == -1


def test_gated_arguments(lib):
    good = dict(type=1, activation=0, N=4, D=16, F=24, x=4096, ldx=16, w_gate=4096, w_up=4096, w_down=4096, b_gate=None, b_up=None, b_down=None)
    for change, code in ((dict(type=3), -2), (dict(activation=3), -2), (dict(N=-1), -1), (dict(D=0), -1), (dict(F=0), -1), (dict(w_up=None), -1),
                         (dict(x=None), -1), (dict(ldx=-1), -1), (dict(N=2 ** 27), -4), (dict(D=70000), -4), (dict(F=2 ** 19), -4)):
        args = lib.GatedFFN(**dict(good, **change))
        assert code_of(lib, "cf_gated_ffn_fwd", ctypes.byref(args), 4096, 4096, None) == code, change
        grads = lib.GatedFFNGrads(4096)
        assert code_of(lib, "cf_gated_ffn_bwd", ctypes.byref(args), ctypes.byref(grads), 4096, None) == code, change
        assert lib.load().cf_gated_ffn_workspace_bytes(ctypes.byref(args), 4096, 1) == 0
    args = lib.GatedFFN(**good)
    assert code_of(lib, "cf_gated_ffn_fwd", ctypes.byref(args), None, 4096, None) == -1
    assert code_of(lib, "cf_gated_ffn_fwd", ctypes.byref(args), 4096, 4096 + 16, None) == -1  # alignment of the workspace
    assert code_of(lib, "cf_gated_ffn_bwd", ctypes.byref(args), None, 4096, None) == -1
    assert code_of(lib, "cf_gated_ffn_bwd", ctypes.byref(args), ctypes.byref(lib.GatedFFNGrads()), 4096, None) == -1
    lib.call("cf_gated_ffn_fwd", ctypes.byref(lib.GatedFFN(**dict(good, N=0, x=None))), None, None, None)


def test_structures_match_the_header(lib):
    """Naturally aligned C structures of 32- and 64-bit fields."""
    assert ctypes.sizeof(lib.QkNorm) == 8 + 7 * 8 + 10 * 8 + 2 * 8 + 8
    assert ctypes.sizeof(lib.GatedFFN) == 8 + 3 * 8 + 2 * 8 + 6 * 8 and ctypes.sizeof(lib.GatedFFNGrads) == 8 * 8


def test_shortest_waves():
    from crystalformer_b200.qk_norm import shortest_waves
    w = shortest_waves(8, 8).reshape(-1, 3)
    every = {tuple(v) for v in w.tolist()}
    assert len(every) == 64 and not any(tuple(-c for c in v) in every for v in every) and all(float(c).is_integer() for v in every for c in v)
    # none left out is shorter than one that is there
    longest = float((w * w).sum(1).max())
    r = range(-4, 5)
    shorter = {v for v in ((a, b, c) for a in r for b in r for c in r) if 0 < sum(i * i for i in v) < longest}
    assert len(shorter) // 2 <= 64


def test_options_of_the_layers():
    from crystalformer_b200.encoder import CrystalformerEncoderLayerCUDA
    from crystalformer_b200.params import LatticeformerParams
    params = LatticeformerParams(qk_norm=True, qk_rotation=8, scale_real=1.4, scale_reci=2.2)
    plain = CrystalformerEncoderLayerCUDA(128, 8, 512, 0.0, "relu", params=LatticeformerParams(scale_real=1.4, scale_reci=2.2))
    layer = CrystalformerEncoderLayerCUDA(128, 8, 512, 0.0, "swiglu", params=params)
    more = set(layer.state_dict()) - set(plain.state_dict())
    assert more == {"linear_gate.weight", "linear_gate.bias", "self_attn.qk_norm.q_weight", "self_attn.qk_norm.k_weight", "self_attn.qk_norm.waves"}
    assert set(plain.state_dict()) <= set(layer.state_dict()) and plain.gate is None and plain.self_attn.qk_norm is None
    assert layer.gate == "silu" and layer.self_attn.qk_norm.waves.shape == (8, 8, 3)


def test_kinds_of_errors(lib):
    """What the torch functions throw arrives as Python's own exceptions."""
    from crystalformer_b200 import ops
    with pytest.raises(ValueError, match="does not belong"):
        ops.embed_bwd(torch.zeros(3, dtype=torch.int64), torch.zeros(4, 8), 5)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.embed_bwd(torch.zeros(4, dtype=torch.int64), torch.zeros(4, 8), 5)
    with pytest.raises(TypeError):
        ops.embed_bwd(None, torch.zeros(4, 8), 5)
    with pytest.raises(ValueError):
        ops.gated_ffn_fwd(torch.zeros(3, 4), torch.zeros(5, 4), torch.zeros(5, 4), torch.zeros(4, 5), activation="tanh")
