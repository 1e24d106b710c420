"""The engine with its projections on the dense operators (fused_dense=True)."""
import pytest
import torch

from helpers import RTOL_BF16, RTOL_FP32, assert_rel, golden, sub
from test_gpu_engine import small_101m_shape
from test_model_host import tiny_config
from maba_v2_architecture_b200 import _native as N
from maba_v2_architecture_b200.engine import MabaEngine, ModelShape, init_state_dict

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_prefill_logits_vs_reference_golden():
    g = golden("model")
    sd = {k: torch.from_numpy(v) for k, v in sub(g, "w.").items()}
    eng = MabaEngine(tiny_config(), sd, dtype=torch.float32, fused_dense=True)
    logits = eng.forward(torch.from_numpy(g["ids"]).to(DEV))
    assert_rel(logits, g["logits"], RTOL_FP32, "engine prefill logits")


@pytest.mark.parametrize("dtype,rtol", [(torch.float32, RTOL_FP32), (torch.bfloat16, RTOL_BF16)])
@pytest.mark.parametrize("B,T", [(2, 150), (1, 7)])
def test_fused_equals_separate_kernels(B, T, dtype, rtol):
    """Against the engine with library products, at the 101M layer shapes (three DGDA blocks, one
    MABA-SA); a decode step after either prefill."""
    cfg = small_101m_shape()
    sd = init_state_dict(ModelShape.from_config(cfg), seed=41)
    ids = torch.randint(0, cfg.vocab_size, (B, T), generator=torch.Generator().manual_seed(42)).to(DEV)
    out = []
    for fused in (False, True):
        eng = MabaEngine(cfg, sd, dtype=dtype, fused_dense=fused)
        logits = eng.forward(ids)
        sess = eng.new_session(batch=B, max_len=T + 8)
        sess.prefill(ids)
        out.append((logits, sess.step(ids[:, 0]).clone()))
    assert_rel(out[1][0], out[0][0], rtol, "prefill")
    assert_rel(out[1][1], out[0][1], rtol, "decode step")
    assert N.device_error() == 0
