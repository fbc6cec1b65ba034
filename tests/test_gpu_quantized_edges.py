"""8-bit pool on the GPU at the edges of what its kernels list and hold."""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import shardserve_b200 as sb
from shardserve_b200 import _native
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


# ---- the workspace ------------------------------------------------------------------------------
FRESH = """
import sys
import torch
sys.path.insert(0, {root!r})
import shardserve_b200 as sb
from shardserve_b200 import kernel as K
k = torch.zeros(4, 16, 2, 128, dtype=torch.int8, device="cuda:0")
v, s = torch.zeros_like(k), torch.ones(4, 2, 2, device="cuda:0")
x = torch.ones(3, 2, 128, device="cuda:0").bfloat16()
q = torch.ones(3, 16, 128, device="cuda:0").bfloat16()
i = torch.zeros(3, dtype=torch.int32, device="cuda:0")
bt = torch.zeros(1, 4, dtype=torch.int32, device="cuda:0")
attend = lambda: sb.ragged_attention_q8(q, k, v, s, bt, i, i, 0.1)
{body}
print("fine")
"""


def fresh_process(body):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = FRESH.format(root=root, body=body)
    run = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and run.stdout.strip() == "fine", run.stderr[-2000:]


@pytest.mark.parametrize("first", ["sb.kv_append_q8(k, v, s, x, x, i + 999)", "sb.kv_read_q8(k, v, s, i + 999)",
                                   "sb.build_block_tables(i - 5, i, bt.expand(3, 4).clone(), i, i[:1], 0)"])
def test_error_bits_outlive_the_first_attention(first):
    """Bits set by the first call of a process are still there after the first attention."""
    bit = _native.SS_DEVERR_POS if "tables" in first else _native.SS_DEVERR_SLOT
    fresh_process(f"{first}\nattend()\nassert K.device_errors(torch.device('cuda:0')) == {bit}")


def test_any_first_call_prepares_a_capture():
    """After an append alone, tables, append, attention and read-back can be captured, and an append's
    bits from inside the graph are seen."""
    fresh_process("""
sb.kv_append_q8(k, v, s, x, x, i)
slots = i + 999
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    sb.build_block_tables(i[:1], i[:1], bt, i, i[:1], 2)
    sb.kv_append_q8(k, v, s, x, x, slots)
    out = attend()
    back = sb.kv_read_q8(k, v, s, i)
graph.replay()
assert torch.equal(out, attend()) and torch.equal(back[0], sb.kv_read_q8(k, v, s, i)[0])
assert K.device_errors(torch.device('cuda:0')) == 8  # SS_DEVERR_SLOT""")
