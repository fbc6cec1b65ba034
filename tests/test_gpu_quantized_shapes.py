"""8-bit attention at the sizes where its kernels change course: rows cut by warps and by CTAs, runs
on both sides of the tiles' shortest run, windows cut over many CTAs, several launches per call.

The plain form is 64-bit torch, row by row; the tolerance is the one of test_gpu_quantized.py
(output rounded to bf16, weights to 11 bits, scores through fp32), asserted doubled."""
import numpy as np
import pytest
import torch

import shardserve_b200 as sb
from shardserve_b200 import kernel as K
from test_gpu_quantized import DEV, batch, dev, make_pool

pytestmark = pytest.mark.gpu


def check(spans, heads, kvh, d, codes, order="head", sm_scale=None, path=None, seed=0):
    sm_scale = d ** -0.5 if sm_scale is None else sm_scale
    pages = sum((c + n + 15) // 16 for c, n in spans) + 3
    k, v, s = make_pool(pages, kvh, d, codes, order, seed=seed)
    tables, seqs, pos, _ = batch(spans, pages, seed=seed)
    g = torch.Generator(device=DEV).manual_seed(seed)
    q = torch.randn(len(seqs), heads, d, device=DEV, generator=g).bfloat16()
    args = (q, k, v, s, dev(tables, torch.int32), dev(seqs, torch.int32), dev(pos, torch.int64), sm_scale)
    K.device_errors(torch.device(DEV))
    out = sb.ragged_attention_q8(*args)
    if path is not None:
        assert K.last_attention_path() == path
    again = sb.ragged_attention_q8(*args)
    assert K.device_errors(torch.device(DEV)) == 0
    assert torch.equal(out, again)
    share = heads // kvh
    t = 0
    for r, (c, n) in enumerate(spans):
        ids = torch.from_numpy(tables[r, :(c + n + 15) // 16]).to(DEV)
        kv = []
        for which, pool in enumerate((k, v)):
            x = pool.contiguous()[ids].float().double() * s[ids][:, None, :, which, None].double()
            kv.append(x.flatten(0, 1)[:c + n].permute(1, 0, 2))            # [kvh, keys, d]
        for a in range(0, n, 512):
            b = min(a + 512, n)
            qq = q[t + a:t + b].double().reshape(b - a, kvh, share, d).permute(1, 2, 0, 3)
            x = qq @ kv[0][:, None].transpose(2, 3) * sm_scale              # [kvh, share, n, keys]
            seen = torch.arange(c + n, device=DEV)[None] <= torch.arange(c + a, c + b, device=DEV)[:, None]
            p = torch.softmax(x.masked_fill(~seen, float("-inf")), -1)
            want = (p @ kv[1][:, None]).permute(2, 0, 1, 3).reshape(b - a, heads, d)
            weight = (p @ kv[1][:, None].abs()).permute(2, 0, 1, 3).reshape(b - a, heads, d)
            got = out[t + a:t + b].double()
            bound = 2 * (2.0 ** -9 * want.abs() + 2.0 ** -10 * weight) + 1e-30
            worst = ((got - want).abs() / bound).max().item()
            assert worst <= 1.0, (r, a, worst)
        t += n


@pytest.mark.parametrize("lo,hi,rows", [(1, 40, 900), (1, 700, 130), (1, 3000, 40), (5000, 9000, 6)])
@pytest.mark.parametrize("codes", ["int8", "e4m3"])
@pytest.mark.parametrize("d,heads,kvh", [(128, 16, 2), (64, 12, 3), (128, 32, 2)])
def test_rows_cut_anywhere(lo, hi, rows, codes, d, heads, kvh):
    rng = np.random.RandomState(rows + d)
    check([(int(n) - 1, 1) for n in rng.randint(lo, hi + 1, rows)], heads, kvh, d, codes, path=5, seed=rows)


@pytest.mark.parametrize("tokens", [6143, 6144, 6145, 12300])
def test_more_rows_than_a_launch_lists(tokens):
    rng = np.random.RandomState(tokens)
    check([(int(n) - 1, 1) for n in rng.randint(1, 60, tokens)], 8, 1, 64, "int8", path=5)


@pytest.mark.parametrize("run", [1, 2, 6, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65])
def test_runs_around_the_shortest_tile(run):
    check([(50, run), (3, 1), (0, run), (400, run), (129, 1), (120, run)], 16, 2, 128, "int8", seed=run)


@pytest.mark.parametrize("group", [1, 2, 3, 4, 5, 7, 8, 12, 16])
@pytest.mark.parametrize("d,codes", [(128, "int8"), (64, "e4m3")])
def test_tiles_of_every_group(group, d, codes):
    check([(0, 300), (77, 140), (200, 9), (31, 1)], 2 * group, 2, d, codes, path=7, seed=group)


@pytest.mark.parametrize("spans", [[(20000, 9)], [(9000, 40), (30, 1), (0, 700)], [(0, 2500)],
                                   [(127, 1000), (128, 8), (0, 8)], [(0, 9)] * 70])
@pytest.mark.parametrize("order", ["head", "token"])
def test_windows_cut_over_ctas(spans, order):
    check(spans, 16, 2, 128, "int8", order, path=7)


@pytest.mark.parametrize("spans", [[(0, 8192)], [(5, 8191), (9, 1)], [(0, 8193)], [(0, 5000), (64, 4000)],
                                   [(0, 8188), (0, 9), (100, 1)]])
def test_prompts_around_a_launch(spans):
    check(spans, 8, 1, 64, "e4m3", path=7)


@pytest.mark.parametrize("sm_scale", [-0.3, 0.0, 0.9])
def test_tiles_scale_signs(sm_scale):
    check([(300, 200), (0, 77)], 16, 2, 128, "e4m3", sm_scale=sm_scale, path=7)


def test_mixed_batch_of_the_benchmark():
    rng = np.random.RandomState(3)
    spans = [(int(c) - 1, 1) for c in rng.randint(256, 4097, 56)] + [(int(c), 512) for c in rng.randint(0, 2049, 8)]
    check(spans, 16, 2, 128, "int8", path=7)


def test_positions_out_of_order_in_a_run():
    """A run's tokens attend to their own positions, whatever their order."""
    k, v, s = make_pool(40, 2, 128, "int8", seed=1)
    tables, seqs, pos, _ = batch([(0, 300)], 40)
    order = np.random.RandomState(0).permutation(300)
    q = torch.randn(300, 16, 128, device=DEV).bfloat16()
    sorted_out = sb.ragged_attention_q8(q, k, v, s, dev(tables, torch.int32), dev(seqs, torch.int32),
                                        dev(pos, torch.int64), 0.1)
    out = sb.ragged_attention_q8(q[torch.from_numpy(order).to(DEV)], k, v, s, dev(tables, torch.int32),
                                 dev(seqs, torch.int32), dev(pos[order], torch.int64), 0.1)
    # Other windows, other orders of summation: both within the tolerance of the same rows.
    diff = (out.double() - sorted_out[torch.from_numpy(order).to(DEV)].double()).abs()
    assert diff.max().item() <= 4 * (2.0 ** -9 + 2.0 ** -10) * float(v.float().abs().max() * s[:, :, 1].max())


@pytest.mark.parametrize("pad", [1, 31, 40])
@pytest.mark.parametrize("kvh", [1, 2, 40])
def test_padding_between_rows(pad, kvh):
    """Padding tokens in the middle of a batch: zero rows, and the others as without them."""
    rng = np.random.RandomState(pad)
    spans = [(int(n) - 1, 1) for n in rng.randint(1, 900, 24)]
    pages = sum((c + n + 15) // 16 for c, n in spans) + 3
    k, v, s = make_pool(pages, kvh, 64, "int8", seed=pad)
    tables, seqs, pos, _ = batch(spans, pages, seed=pad)
    q = torch.randn(len(seqs) * (pad + 1), 2 * kvh, 64, device=DEV).bfloat16()
    real = torch.arange(len(seqs), device=DEV) * (pad + 1) + pad // 2
    wide_seqs = torch.full((len(q),), -1, dtype=torch.int32, device=DEV)
    wide_pos = torch.full((len(q),), -1, dtype=torch.int64, device=DEV)
    wide_seqs[real], wide_pos[real] = dev(seqs, torch.int32), dev(pos, torch.int64)
    bt = dev(tables, torch.int32)
    K.device_errors(torch.device(DEV))
    out = sb.ragged_attention_q8(q, k, v, s, bt, wide_seqs, wide_pos, 0.125)
    alone = sb.ragged_attention_q8(q[real], k, v, s, bt, dev(seqs, torch.int32), dev(pos, torch.int64), 0.125)
    assert K.device_errors(torch.device(DEV)) == 0
    assert not out[wide_seqs == -1].any()
    # Other shares of the warps, other orders of summation: both within the tolerance of the same rows.
    diff = (out[real].double() - alone.double()).abs().max().item()
    assert diff <= 4 * (2.0 ** -9 + 2.0 ** -10) * float(v.float().abs().max() * s[:, :, 1].max())
