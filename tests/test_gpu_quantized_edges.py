"""8-bit pool on the GPU at the edges of what its kernels list and hold."""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import shardserve_b200 as sb
from shardserve_b200 import _native
from shardserve_b200 import kernel as K
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


@pytest.mark.parametrize("cols,path", [(16_700_000, 7), (16_770_000, 5)])
def test_tables_too_wide_for_a_launch_of_tiles(cols, path):
    """1025 windows of the widest table whose blocks the tiles count in 31 bits, and of a wider one."""
    k, v, s = make_pool(4, 1, 64, "int8")
    tables = torch.zeros((1, cols), dtype=torch.int32, device=DEV)
    tables[0, :2] = torch.tensor([3, 1], dtype=torch.int32, device=DEV)
    q = torch.randn(20, 4, 64, device=DEV).bfloat16()
    seqs, pos = np.zeros(20, np.int64), np.arange(5, 25)
    out = sb.ragged_attention_q8(q, k, v, s, tables, dev(seqs, torch.int32), dev(pos, torch.int64), 0.1)
    assert K.last_attention_path() == path
    check_attention(out, q, k, v, s, np.array([[3, 1]]), seqs, pos, 0.1)


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


# ---- NaN codes --------------------------------------------------------------------------------
def nan_case(order="head", d=128, heads=16, kvh=2, spans=((200, 40), (3, 1), (0, 300)), seed=13):
    pages = sum((c + n + 15) // 16 for c, n in spans) + 2
    k, v, s = make_pool(pages, kvh, d, "e4m3", order, seed=seed)
    tables, seqs, pos, _ = batch(spans, pages, seed=seed)
    g = torch.Generator(device=DEV).manual_seed(seed)
    q = torch.randn(len(seqs), heads, d, device=DEV, generator=g).bfloat16()
    return q, k, v, s, tables, seqs, pos


@pytest.mark.parametrize("key", list(range(195, 220)) + [0, 131, 239])
def test_nan_key_reaches_the_tokens_that_attend_it(key):
    """One NaN among a K row's codes: the outputs of the tokens that attend the row, in the heads that
    share its KV head, are NaN; every other output keeps its bits."""
    q, k, v, s, tables, seqs, pos = nan_case()
    args = (dev(tables, torch.int32), dev(seqs, torch.int32), dev(pos, torch.int64), 0.1)
    clean = sb.ragged_attention_q8(q, k, v, s, *args)
    k.view(torch.uint8)[tables[0, key // 16], key % 16, 1, 77] = 0x7f
    out = sb.ragged_attention_q8(q, k, v, s, *args)
    hit = torch.zeros(out.shape, dtype=torch.bool, device=DEV)
    hit[:, 8:] = dev((seqs == 0) & (pos >= key), torch.bool)[:, None, None]
    assert torch.isnan(out[hit]).all()
    assert torch.equal(out[~hit], clean[~hit])


@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("heads,kvh", [(16, 2), (32, 2), (48, 2)])
@pytest.mark.parametrize("key", [0, 77, 238, 239])
def test_nan_codes_reach_single_tokens(which, heads, kvh, key):
    """The same for decode rows: the token that attends the row, and no other row."""
    q, k, v, s, tables, seqs, pos = nan_case(heads=heads, spans=((238, 1), (3, 1), (500, 1)))
    args = (dev(tables, torch.int32), dev(seqs, torch.int32), dev(pos, torch.int64), 0.1)
    clean = sb.ragged_attention_q8(q, k, v, s, *args)
    (k if which == "k" else v).view(torch.uint8)[tables[0, key // 16], key % 16, 1, 77] = 0x7f
    out = sb.ragged_attention_q8(q, k, v, s, *args)
    hit = torch.zeros(out.shape, dtype=torch.bool, device=DEV)
    if key < 239:
        hit[0, heads // 2:, 77 if which == "v" else slice(None)] = True
    assert torch.isnan(out[hit]).all()
    assert torch.equal(out[~hit], clean[~hit])


@pytest.mark.parametrize("key", [0, 100, 130, 199, 200, 201, 215, 220, 231, 239])
@pytest.mark.parametrize("order,d,heads,kvh", [("head", 128, 16, 2), ("token", 64, 2, 2), ("head", 64, 14, 2)])
def test_nan_value_reaches_the_tokens_that_attend_it(key, order, d, heads, kvh):
    """NaN codes in a V row: the outputs of the tokens that attend the row are NaN in those places
    of head_dim and no others; tokens before the row do not see it."""
    q, k, v, s, tables, seqs, pos = nan_case(order, d, heads, kvh)
    args = (dev(tables, torch.int32), dev(seqs, torch.int32), dev(pos, torch.int64), 0.1)
    clean = sb.ragged_attention_q8(q, k, v, s, *args)
    places = [5, 16, 31, 33, d - 1]
    raw = v.view(torch.uint8)
    raw[tables[0, key // 16], key % 16, 1, places] = torch.tensor([0x7f, 0xff, 0x7f, 0xff, 0x7f], dtype=torch.uint8, device=DEV)
    out = sb.ragged_attention_q8(q, k, v, s, *args)
    hit = torch.zeros(out.shape, dtype=torch.bool, device=DEV)
    rows = dev((seqs == 0) & (pos >= key), torch.bool)
    for p in places:
        hit[:, heads // 2:, p] = rows[:, None]
    assert torch.isnan(out[hit]).all()
    assert torch.equal(out[~hit], clean[~hit])


@pytest.mark.parametrize("spans", [[(200, 40), (0, 300)], [(239, 1), (299, 1)]])
def test_nan_value_in_a_page_of_zeros(spans):
    """A page whose V scale is 0, with one NaN among its codes: NaN times any scale is NaN, in the tiles and
    in the split-K kernel."""
    q, k, v, s, tables, seqs, pos = nan_case(spans=spans)
    args = (dev(tables, torch.int32), dev(seqs, torch.int32), dev(pos, torch.int64), 0.1)
    s[tables[0, 3], 1, 1] = 0.0
    clean = sb.ragged_attention_q8(q, k, v, s, *args)
    v.view(torch.uint8)[tables[0, 3], 4, 1, 70] = 0xff
    out = sb.ragged_attention_q8(q, k, v, s, *args)
    hit = torch.zeros(out.shape, dtype=torch.bool, device=DEV)
    hit[:, 8:, 70] = dev(seqs == 0, torch.bool)[:, None]
    assert torch.isnan(out[hit]).all()
    assert torch.equal(out[~hit], clean[~hit])


def test_nan_values_where_a_window_is_cut():
    """A run of positions in no order over a long context, cut over many CTAs: NaN codes of V at both
    ends and in the middle reach the tokens at or past them alone."""
    q, k, v, s, tables, seqs, pos = nan_case(spans=((6000, 32), (0, 40)))
    pos = pos.copy()
    pos[:32] = np.random.RandomState(5).randint(0, 6032, 32)
    args = (dev(tables, torch.int32), dev(seqs, torch.int32), dev(pos, torch.int64), 0.1)
    clean = sb.ragged_attention_q8(q, k, v, s, *args)
    raw = v.view(torch.uint8)
    hit = torch.zeros(clean.shape, dtype=torch.bool, device=DEV)
    for key, place in ((17, 3), (2999, 64), (3000, 65), (6030, 127)):
        raw[tables[0, key // 16], key % 16, 0, place] = 0x7f
        hit[:, :8, place] = dev((seqs == 0) & (pos >= key), torch.bool)[:, None]
    out = sb.ragged_attention_q8(q, k, v, s, *args)
    assert torch.isnan(out[hit]).all()
    assert torch.equal(out[~hit], clean[~hit])


# ---- infinities in the append ---------------------------------------------------------------------
@pytest.mark.parametrize("codes", ["int8", "e4m3"])
@pytest.mark.parametrize("rest", [0.0, 1e-35, 0.75])
def test_infinities_saturate_beside_any_values(codes, rest):
    """An infinity takes the largest code's place whatever stands beside it; where nothing finite does, the
    scale is 0 and so is every value.  NaN stays NaN in e4m3 and becomes 0 in int8."""
    k, v, s = (t.clone() for t in make_pool(3, 1, 64, codes, seed=3))
    x = torch.full((4, 1, 64), rest, device=DEV)
    x[1, 0, 5], x[2, 0, 6] = float("inf"), float("-inf")
    nan = x.clone()
    nan[3, 0, 7] = float("nan")
    sb.kv_append_q8(k, v, s, x.bfloat16(), nan.bfloat16(), dev(range(16, 20), torch.int64))
    rk, rv = sb.kv_read_q8(k, v, s, dev(range(16, 20), torch.int64))
    top = float(torch.tensor(rest).bfloat16()) if rest == 0.75 else 0.0
    want = torch.full((4, 1, 64), top, device=DEV)
    want[2, 0, 6] = -top
    assert torch.allclose(rk.float(), want, rtol=2.0 ** -7, atol=0.0)
    if codes == "int8":
        want[3, 0, 7] = 0.0
    else:
        assert rv[3, 0, 7].isnan()
        rv[3, 0, 7] = want[3, 0, 7]
    assert torch.allclose(rv.float(), want, rtol=2.0 ** -7, atol=0.0)


# ---- weights of the tiles ---------------------------------------------------------------------
@pytest.mark.parametrize("codes", ["int8", "e4m3"])
@pytest.mark.parametrize("spans", [[(300, 1)] * 40, [(300, 64)]])
def test_outputs_are_not_biased(codes, spans):
    """The weights are rounded to nearest before the product with V, whose sum l does not see.  An
    output's own rounding (half of 2^-8) averages out over the 81,920 or more outputs, a weight's (2^-12)
    over the 300 keys too; what is left of the outputs' common factor is below 2^-14.  (Weights cut
    off at tf32's 11 bits would make it 1 - 2^-11 * 0.7.)"""
    heads, kvh, d = 16, 2, 128
    k, v, s = make_pool(40 * 19 + 30, kvh, d, codes, seed=12)
    tables, seqs, pos, _ = batch(spans, 40 * 19 + 30, seed=12)
    g = torch.Generator(device=DEV).manual_seed(12)
    q = torch.randn(len(seqs), heads, d, device=DEV, generator=g).bfloat16()
    out = sb.ragged_attention_q8(q, k, v, s, dev(tables, torch.int32), dev(seqs, torch.int32),
                                 dev(pos, torch.int64), 0.09)
    want = check_attention(out, q, k, v, s, tables, seqs, pos, 0.09)
    factor = (out.cpu().double().numpy() * want).sum() / (want * want).sum()
    assert abs(factor - 1) < 2.0 ** -14, factor - 1


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


# ---- inputs that the kernel before the call writes -----------------------------------------------
@pytest.mark.parametrize("last", ["tables", "positions", "ids"])
@pytest.mark.parametrize("chunk", [1, 40])
def test_inputs_written_by_the_kernel_before(last, chunk):
    """The kernel right before the attention writes its tables, positions or ids, with nothing between:
    every call sees that step's values."""
    rows, steps = 48, 30
    spans = [(13 * r % 700, chunk) for r in range(rows)]
    pages = sum((c + n + 15) // 16 for c, n in spans) + 3
    k, v, s = make_pool(pages, 2, 128, "int8", seed=21)
    tables, seqs, pos, _ = batch(spans, pages, seed=21)
    rng = np.random.RandomState(0)
    sets = []
    for _ in range(3):  # the same rows in another order
        order = rng.permutation(rows)
        place = np.argsort(order)
        sets.append([dev(tables[order], torch.int32), dev(place[seqs], torch.int32), dev(pos, torch.int64)])
    sets.append([sets[0][0], sets[0][1], dev(pos // 2, torch.int64)])
    q = torch.randn(len(seqs), 16, 128, device=DEV).bfloat16()
    want = [sb.ragged_attention_q8(q, k, v, s, *x, 0.1) for x in sets]
    now = [x.clone() for x in sets[0]]
    at = {"tables": 0, "ids": 1, "positions": 2}[last]
    got = []
    for i in range(steps):
        one = sets[i * 7 % 4]
        for j in (0, 1, 2):
            if j != at:
                now[j].copy_(one[j])
        now[at].copy_(one[at])
        got.append(sb.ragged_attention_q8(q, k, v, s, *now, 0.1))
    for i, x in enumerate(got):
        assert torch.equal(x, want[i * 7 % 4]), i


def test_tables_right_before_the_attention():
    """build_block_tables, then the attention with nothing between, over rows that grow by one token."""
    rows, steps = 40, 25
    cached = np.array([9 * r % 200 for r in range(rows)])
    k, v, s = make_pool(rows * 16, 2, 64, "e4m3", seed=22)
    tables = np.arange(rows * 16).reshape(rows, 16)  # every row's pages are known beforehand
    lens, new = dev(cached, torch.int32), torch.ones(rows, dtype=torch.int32, device=DEV)
    bt, head = dev(tables, torch.int32), torch.zeros(1, dtype=torch.int32, device=DEV)
    # The free list holds, in the order in which they are taken, the pages that stand there already.
    taken = [tables[r, (cached[r] + t) // 16] for t in range(steps) for r in range(rows) if (cached[r] + t) % 16 == 0]
    q = torch.randn(rows, 16, 64, device=DEV).bfloat16()
    got = []
    free = dev(taken, torch.int32)
    for _ in range(steps):
        m = sb.build_block_tables(lens, new, bt, free, head, rows, out={"lens": lens, "free_head": head})
        got.append(sb.ragged_attention_q8(q, k, v, s, m["tables"], m["seqs"], m["positions"], 0.1))
    for t, out in enumerate(got):
        want = sb.ragged_attention_q8(q, k, v, s, dev(tables, torch.int32), dev(np.arange(rows), torch.int32),
                                      dev(cached + t, torch.int64), 0.1)
        assert torch.equal(out, want), t
    assert int(head) == len(taken)


# ---- lengths past any table ----------------------------------------------------------------------
@pytest.mark.parametrize("cached,new", [([3, 3, 3, 3], [2 ** 62] * 4), ([2 ** 63 - 1, 5, 0, 0], [2 ** 63 - 1, 2, 1, 1]),
                                        ([0, 2 ** 62, 1, 0], [1, 2, 2 ** 63 - 1, 1])])
def test_block_tables_lengths_near_64_bits(cached, new):
    """Sums of such lengths pass 64 bits: the first rows' tokens stand where they belong, lengths saturate,
    nothing past a table gets a slot, and the error bit is set."""
    tokens, width = 6, 2
    free = np.arange(50, 70)
    K.device_errors(torch.device(DEV))
    tables = torch.arange(8, device=DEV).reshape(4, width)
    got = sb.build_block_tables(torch.tensor(cached, device=DEV), torch.tensor(new, device=DEV), tables,
                                dev(free, torch.int64), torch.zeros(1, dtype=torch.int32, device=DEV), tokens)
    assert K.device_errors(torch.device(DEV)) & _native.SS_DEVERR_POS
    seqs, pos, slots, last = [], [], [], [-1] * 4
    table, taken = np.arange(8).reshape(4, width), 0
    for r in range(4):
        for col in range((cached[r] + 15) // 16, min((cached[r] + new[r] + 15) // 16, width)):
            table[r, col] = free[taken]
            taken += 1
    for r in range(4):
        for p in range(cached[r], cached[r] + min(new[r], tokens)):
            if len(seqs) < tokens:
                last[r] = len(seqs)
                seqs.append(r)
                pos.append(p)
                slots.append(int(table[r, p // 16]) * 16 + p % 16 if p < 16 * width else -1)
    assert got["seqs"].tolist() == seqs
    assert got["slots"].tolist() == slots
    if max(cached) < 2 ** 61:
        assert got["positions"].tolist() == pos
    assert got["last"].tolist() == last
    assert got["lens"].tolist() == [min(c + n, 2 ** 31 - 1) for c, n in zip(cached, new)]
    assert got["tables"].cpu().numpy().tolist() == table.tolist()
    assert int(got["free_head"]) == taken
