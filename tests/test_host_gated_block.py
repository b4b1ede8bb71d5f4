"""Arguments that the entry points of the gated block refuse before they touch a GPU."""
import ctypes

import pytest
import torch

import torchgt_amd as T
from torchgt_amd import _lib

BAD, UNSUPPORTED, OK, WORKSPACE = _lib.ERR_INVALID_ARG, _lib.ERR_UNSUPPORTED, _lib.OK, _lib.ERR_WORKSPACE


def test_entry_points_refuse_bad_arguments():
    L = _lib.lib()
    p = ctypes.c_void_p(4096)      # (never read: every call below ends before a launch)
    assert L.tgt_gated_linear_fwd(p, p, p, None, None, -1, 8, 8, 0, 3, p, None, None, 0, None) == BAD
    assert L.tgt_gated_linear_fwd(p, p, p, None, None, 4, 0, 8, 0, 3, p, None, None, 0, None) == BAD
    assert L.tgt_gated_linear_fwd(p, p, p, None, None, 4, 8, 8, 2, 3, p, None, None, 0, None) == BAD          # dtype
    assert L.tgt_gated_linear_fwd(p, p, p, None, None, 4, 8, 8, 0, 4, p, None, None, 0, None) == BAD          # activation
    assert L.tgt_gated_linear_fwd(None, p, p, None, None, 4, 8, 8, 0, 3, p, None, None, 0, None) == BAD
    assert L.tgt_gated_linear_fwd(p, p, None, None, None, 4, 8, 8, 0, 3, p, None, None, 0, None) == BAD
    assert L.tgt_gated_linear_fwd(p, p, p, None, None, 4, 8, 8, 0, 3, None, None, None, 0, None) == BAD
    assert L.tgt_gated_linear_fwd(p, p, p, None, None, 1 << 31, 8, 8, 0, 3, p, None, None, 0, None) == UNSUPPORTED
    assert L.tgt_gated_linear_fwd(None, None, None, None, None, 0, 8, 8, 0, 3, None, None, None, 0, None) == OK          # nothing to do
    assert L.tgt_linear_epilogue_fwd(p, None, None, None, 4, 8, 8, 0, 0, p, None, None, 0, None) == BAD
    assert L.tgt_linear_epilogue_8bit_fwd(p, p, p, p, None, None, 4, 24, 8, 0, 0, p, None, 0, None) == UNSUPPORTED
    assert L.tgt_linear_epilogue_8bit_fwd(p, None, p, p, None, None, 4, 32, 8, 0, 0, p, None, 0, None) == BAD
    assert L.tgt_gated_linear_8bit_fwd(p, p, p, p, p, None, None, None, 4, 32, 8, 0, 0, p, None, 0, None) == BAD
    for fwd, lead in (("tgt_gated_linear", (p, p, p, None, None)), ("tgt_linear_epilogue", (p, p, None, None))):      # few rows, a long contraction: cut in pieces
        need = getattr(L, fwd + "_fwd_workspace_bytes")(300, 4096, 512, 1)
        assert need > 0 and getattr(L, fwd + "_fwd_workspace_bytes")(64, 4096, 512, 1) == 0 == getattr(L, fwd + "_fwd_workspace_bytes")(0, 4096, 512, 1)
        assert getattr(L, fwd + "_fwd_workspace_bytes")(-1, 4096, 512, 1) == -1 and getattr(L, fwd + "_8bit_workspace_bytes")(5, 0, 512) == -1
        call = getattr(L, fwd + "_fwd")
        assert call(*lead, 300, 4096, 512, 1, 3, p, None, p, 1024, None) == WORKSPACE and call(*lead, 300, 4096, 512, 1, 3, p, None, None, need, None) == WORKSPACE
        assert call(*lead, 300, 4096, 512, 1, 3, p, None, ctypes.c_void_p(4100), need, None) == WORKSPACE
    assert L.tgt_linear_epilogue_8bit_fwd(p, p, p, p, None, None, 300, 4096, 512, 1, 0, p, None, 0, None) == WORKSPACE
    dW = (ctypes.c_void_p * 2)(4096, None)
    assert L.tgt_gated_linear_bwd(p, p, p, None, None, p, 4, 8, 8, 0, 3, None, p, dW, None, p, 1 << 20, None) == BAD      # one weight's gradient
    assert L.tgt_gated_linear_bwd(p, p, p, None, None, None, 4, 8, 8, 0, 3, None, p, None, None, p, 1 << 20, None) == BAD
    assert L.tgt_gated_linear_bwd(p, p, p, None, None, p, 4, 8, 8, 0, 3, None, p, None, None, None, 0, None) == WORKSPACE
    need = L.tgt_gated_linear_bwd_workspace_bytes(1000, 64, 128, 0)
    assert need >= 1000 * 256 * 4
    assert L.tgt_gated_linear_bwd(p, p, p, None, None, p, 1000, 64, 128, 0, 3, None, p, None, None, p, need - 16, None) == WORKSPACE
    assert L.tgt_gated_linear_bwd(p, p, p, None, None, p, 1000, 64, 128, 0, 3, None, p, None, None, ctypes.c_void_p(4100), need, None) == WORKSPACE
    assert L.tgt_gated_linear_bwd_workspace_bytes(-1, 64, 128, 0) == -1 and L.tgt_gated_linear_bwd_workspace_bytes(5, 64, 128, 7) == -1
    assert L.tgt_linear_epilogue_bwd_workspace_bytes(5, 0, 128, 0, 0) == -1
    assert L.tgt_add_rms_norm_fwd(p, None, p, 4, 0, 1e-6, 0, None, p, None, None) == BAD
    assert L.tgt_add_rms_norm_fwd(p, None, p, 4, 16385, 1e-6, 0, None, p, None, None) == UNSUPPORTED
    assert L.tgt_add_rms_norm_fwd(p, p, p, 4, 64, 1e-6, 0, None, p, None, None) == BAD          # a residual and nowhere to put the sum
    assert L.tgt_add_rms_norm_8bit(p, None, p, 4, 64, 1e-6, 0, None, p, None, None) == BAD
    assert L.tgt_quantize_rows(p, 4, 64, 2, p, p, None) == BAD
    assert L.tgt_quantize_rows(None, 0, 64, 0, None, None, None) == OK
    assert L.tgt_rms_norm_bwd(p, p, p, p, None, 4, 64, 0, p, p, None, 0, None) == WORKSPACE
    assert L.tgt_rms_norm_bwd(p, p, p, p, None, 4, 64, 0, p, None, p, 1 << 20, None) == BAD
    assert L.tgt_rms_norm_bwd_workspace_bytes(4, 64) == 4 * 64 * 4 and L.tgt_rms_norm_bwd_workspace_bytes(-1, 64) == -1


def test_operators_need_a_gpu():
    x, w, v = torch.zeros(4, 16), torch.zeros(8, 16), torch.zeros(16)
    c, s = torch.zeros(4, 16, dtype=torch.float8_e4m3fn), torch.zeros(4)
    for call in (lambda: T.gated_linear(x, w, w), lambda: T.linear_act(x, w), lambda: T.add_rms_norm(x, None, v), lambda: T.add_rms_norm_8bit(x, None, v),
                 lambda: T.quantize_rows(x), lambda: T.linear_act_8bit(c, s, c, s), lambda: T.gated_linear_8bit(c, s, c, s, c, s)):
        with pytest.raises(RuntimeError, match="GPU"):
            call()
    with pytest.raises(ValueError, match="activation"):
        T.linear_act(x, w, activation="tanh")


def test_gated_graphormer_has_its_modules():
    m = T.Graphormer(2, 4, 16, 32, 7, 1, 0.0, 0.0, 0.0, 64, 1, gated=True)
    names = {k for k, _ in m.named_parameters()}
    assert "layers.1.ffn.gate.weight" in names and "layers.0.self_attention_norm.weight" in names and "final_ln.weight" in names
    assert "final_ln.bias" not in names
    assert not T.Graphormer(1, 4, 16, 32, 7, 1, 0.0, 0.0, 0.0, 64, 1).gated
