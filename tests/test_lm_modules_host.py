"""GatedSSM and the options of TSRNTropicalPath on a host without a GPU: parameters, refusals, and
the token models' embedding on the CPU as before."""
import math

import pytest
import torch


def test_gated_ssm_parameters_and_memories():
    from mk_iii_technologies_tsrn_b200.ssm import GatedSSM
    m = GatedSSM(16, 8)
    assert set(m.state_dict()) == {"gate.weight", "gate.bias", "B_proj.weight", "C_proj.weight",
                                   "gate_out.weight", "gate_out.bias", "mix"}
    f = torch.sigmoid(m.gate.bias)
    assert torch.all(f[1:] > f[:-1]) and 0.49 < float(f[0]) < 0.51 and float(f[-1]) > 0.998
    assert torch.all(m.C_proj.weight == 0) and m.init_state(3).shape == (3, 8)
    for grad in (False, True):
        with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="no CPU fallback"):
            m(torch.randn(2, 5, 16))


def test_path_options_keep_the_blocks_names():
    from mk_iii_technologies_tsrn_b200.tsrn_block import TSRNTropicalPath
    plain = TSRNTropicalPath(16, top_k=4, n_heads=2)
    fused = TSRNTropicalPath(16, top_k=4, n_heads=2, fused_residual=True)
    assert set(plain.state_dict()) == set(fused.state_dict())
    fused.load_state_dict(plain.state_dict())
    gated = TSRNTropicalPath(16, top_k=4, n_heads=2, ssm="gated")
    assert "tropical_ssm.gate.weight" in gated.state_dict()
    with pytest.raises(ValueError, match="ssm"):
        TSRNTropicalPath(16, top_k=4, n_heads=2, ssm="linear")


def test_token_embedding_on_the_cpu_is_the_plain_expression():
    from mk_iii_technologies_tsrn_b200 import dropin
    m = dropin.TropicalDecoderModel(11, d_model=8, nhead=2, num_layers=1, dim_feedforward=16,
                                    dropout=0.0, max_seq_len=6)
    ids = torch.randint(0, 11, (2, 6))
    want = m.embed(ids) * math.sqrt(8) + m.pos_embed(torch.arange(6))[None]
    assert torch.equal(m._embed(ids), want)
