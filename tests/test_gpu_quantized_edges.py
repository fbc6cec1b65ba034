"""8-bit pool on the GPU at the edges of what its kernels list and hold."""
import numpy as np
import pytest
import torch

import shardserve_b200 as sb
from test_gpu_quantized import DEV, batch, check_attention, dev, make_pool
from test_gpu_quantized_shapes import check

pytestmark = pytest.mark.gpu


# ---- launches that list the most windows --------------------------------------------------------
@pytest.mark.parametrize("lead,heads,kvh,d", [(1, 8, 1, 64), (3, 2, 2, 64), (7, 16, 1, 128)])
def test_most_windows_of_a_launch(lead, heads, kvh, d):
    """Runs of 8 tokens behind `lead` tokens of another: a launch of 8192 tokens begins and ends inside
    a run, and lists 1025 windows.  Every row against the plain form."""
    runs = 2048 if lead == 1 else 1030
    spans = [(c % 37, 8) for c in range(runs)]
    check([(5, lead)] + spans, heads, kvh, d, "int8", path=7, seed=lead)
    # With two launches' ends inside runs, and runs of other lengths between them.
    mixed = [(c % 29, 8 if c % 7 else 9) for c in range(1200)]
    check([(5, lead)] + mixed, heads, kvh, d, "int8", path=7, seed=lead + 1)


# ---- queries at both ends of bf16's range -----------------------------------------------------
@pytest.mark.parametrize("exponent", [-133, -130, -126, -112, -105, -64, -63, 0, 126, 127])
@pytest.mark.parametrize("codes,heads,kvh", [("int8", 16, 2), ("int8", 16, 1), ("e4m3", 4, 2),
                                             ("int8", 24, 1)])
def test_query_exponents(exponent, codes, heads, kvh):
    """Query rows whose largest value has this exponent, up to bf16's largest finite numbers and
    down to its subnormals, of both signs, with finite scores: decode rows and a prompt chunk."""
    k, v, s = make_pool(40, kvh, 128, codes, seed=6)
    spans = [(60, 1), (170, 1), (10, 40)]
    tables, seqs, pos, _ = batch(spans, 40)
    g = torch.Generator(device=DEV).manual_seed(exponent + 200)
    mantissa = 1 + torch.randint(0, 128, (len(seqs), heads, 128), device=DEV, generator=g) / 128.0
    sign = 1.0 - 2.0 * torch.randint(0, 2, mantissa.shape, device=DEV, generator=g)
    q = (mantissa * sign).cpu().double().numpy() * 2.0 ** exponent
    q = torch.from_numpy(q).float().bfloat16().to(DEV)  # exact, but for subnormals' lost bits
    assert torch.isfinite(q.float()).all() and q.float().abs().min() > 0
    # K's scales and sm_scale together bring the scores to the usual size; each is a normal number.
    up = max(-120, min(120, -exponent))
    s[:, :, 0] *= 2.0 ** (-exponent - up)
    sm_scale = float(np.float32(0.05) * np.float32(2.0 ** up))
    out = sb.ragged_attention_q8(q, k, v, s, dev(tables, torch.int32), dev(seqs, torch.int32),
                                 dev(pos, torch.int64), sm_scale)
    check_attention(out, q, k, v, s, tables, seqs, pos, sm_scale)
