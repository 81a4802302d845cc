"""Beam search's selection on the GPU against the definition in 64 bits."""

import math

import pytest
import torch

from kvserve_amd import paged

from _shared_ref import score_bound, select

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def check(logits, scores, beams, count=None, end=None, **kw):
    got = paged.select_beams(logits, scores, beams, count, end_token=end, **kw)
    n = got.all_parents.shape[1]
    want = select(logits, scores, beams, n, end)
    for k in (0, 1, 3, 4):
        assert torch.equal(got[k].cpu(), want[k]), (k, got[k].cpu(), want[k])
    for k in (2, 5):
        g, w = got[k].cpu().double(), want[k]
        fine = torch.isfinite(w)
        assert torch.equal(g[~fine], w[~fine])
        assert bool(((g - w).abs() <= score_bound(w))[fine].all())
    return got


def rand_logits(dev, rows, V, dtype, seed, pad=0, scale=2.5):
    gen = torch.Generator(device=dev).manual_seed(seed)
    x = (torch.randn((rows, V + pad), generator=gen, device=dev) * scale).to(dtype)[:, :V]
    s = -20.0 * torch.rand(rows, generator=gen, device=dev)
    return x, s


# vocabularies around a vector, a wave, and the ends of tiles of one to eight vectors a thread
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("V", [1, 2, 7, 8, 9, 63, 64, 65, 511, 1000, 1023, 1024, 1025, 2047, 2048, 2049, 4096, 4103, 8192,
                               16383, 16384, 16385, 50021])
def test_vocabularies(cuda, dtype, V):
    x, s = rand_logits(cuda, 6, V, DTYPES[dtype], V)
    check(x, s, 3, 6, end=V // 2)


@pytest.mark.parametrize("beams,count", [(1, 1), (1, 2), (2, 4), (4, 9), (5, 11), (16, 32), (32, 64), (64, 64), (1, 64),
                                         (7, 63)])
def test_beams_and_counts(cuda, beams, count):
    x, s = rand_logits(cuda, 2 * beams, 5000, torch.bfloat16, count)
    check(x, s, beams, count)
    check(x, s, beams, count, end=int(x[0].float().argmax()))


# enough rows that a thread takes 2, 4, 8 and 16 vectors, in rows that begin off the 16-byte places
@pytest.mark.parametrize("dtype,rows,V,pad", [("bf16", 96, 40001, 0), ("bf16", 160, 70000, 3), ("bf16", 192, 100003, 1),
                                              ("fp16", 128, 70001, 0), ("fp32", 32, 70001, 0), ("fp32", 96, 60001, 2),
                                              ("fp32", 128, 70000, 0), ("bf16", 504, 100003, 0),
                                              ("fp32", 256, 98400, 8)])
def test_many_rows(cuda, dtype, rows, V, pad):
    x, s = rand_logits(cuda, rows, V, DTYPES[dtype], rows, pad)
    check(x, s, 4, 8, end=5)


def test_views(cuda):
    """Rows of a larger tensor, every other row, one row for all beams, and a base off by one element."""
    x, s = rand_logits(cuda, 8, 3001, torch.bfloat16, 1)
    check(x[2:6], s[2:6], 2, 4)
    check(x[::2], s[:4], 4, 8)
    check(x[:1].expand(4, -1), s[:4], 4, 8)
    flat = torch.randn(4 * 999 + 1, device=cuda).half()
    check(flat[1:].view(4, 999), s[:4], 2, 5)
    check(x[:, 5:1005], s, 4, 4)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_ties(cuda, dtype):
    """Equal logits everywhere, by plateaus, and equal beams: the lower beam, then the lower token."""
    dt = DTYPES[dtype]
    x = torch.zeros((4, 40000), device=cuda, dtype=dt)
    s = torch.tensor([-1.0, -1.0, -1.0, -1.0], device=cuda)
    got = check(x, s, 2, 64)
    assert got.all_tokens[0].tolist() == list(range(64)) and got.all_parents[1].tolist() == [2] * 64
    x[:, ::2] = -0.0  # the same value as 0
    assert check(x, s, 2, 64).all_tokens[0].tolist() == list(range(64))
    gen = torch.Generator(device=cuda).manual_seed(3)
    x = torch.randint(-2, 3, (4, 40000), generator=gen, device=cuda).to(dt)
    check(x, s, 2, 33, end=int((x[0] == 2).nonzero()[0]))
    x[1], x[3] = x[0], x[2]  # beams alike
    got = check(x, s, 2, 64)
    assert set(got.all_parents[0].tolist()) == {0}
    # 700 equal logits at the border of the best, all of them in a few threads' vectors
    x = torch.randn((2, 30000), generator=gen, device=cuda).to(dt)
    x[0, :1400] = 9.0
    x[1, 2000:2004] = 11.0
    x[1, 29000:] = 10.0
    check(x, torch.tensor([-1.0, -0.5], device=cuda), 2, 50)


def test_large_ones_in_few_threads(cuda):
    """More elements above the bound than a workgroup ranks at once."""
    for dtype in DTYPES.values():
        x = torch.zeros((1, 16384 * 2), device=cuda)
        up = torch.arange(16384 * 2, device=cuda)
        x[0] = torch.where((up // 8) % 64 < 20, 5.0 + (up % 1777).float() / 256, -1.0)
        for rows in (1, 128):
            check(x.to(dtype).expand(rows, -1), torch.linspace(-1, -2, rows, device=cuda), 1, 64)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_masked_vocabularies(cuda, dtype):
    dt = DTYPES[dtype]
    low = torch.finfo(dt).min
    x, s = rand_logits(cuda, 8, 9000, dt, 5)
    for value in (-math.inf, low):
        y = x.clone()
        y[:, 1::2] = value
        y[1] = value                   # a beam with nothing allowed
        y[2, :] = value
        y[2, 77] = 1.0                 # and one with a single token
        y[4:6] = value                 # a whole request
        got = check(y, s, 2, 9, end=77)
        if value == -math.inf:
            assert got.all_parents[2].tolist() == [-1] * 9 and got.parents[4:6].tolist() == [-1, -1]
    # fewer candidates than asked for
    y = torch.full((4, 600), -math.inf, device=cuda, dtype=dt)
    y[0, 3], y[1, 3], y[1, 599] = 1.0, 2.0, 1.5
    got = check(y, s[:4], 4, 8, end=3)
    assert got.tokens.tolist() == [599, -1, -1, -1]


def test_far_logits(cuda):
    """Logits whose exponentials leave 64 bits: sums go by their largest."""
    x, s = rand_logits(cuda, 8, 20000, torch.float32, 6)
    x[0] += 1e4
    x[1] -= 1e4
    x[2] = x[2] * 1e30
    x[3] = x[3] * 300.0
    x[4, 100] = 3e38
    x[5] = torch.finfo(torch.float32).min
    x[6, 5000:] = -1e5   # whole tiles far below the others
    x[7, :5000] = 650.0
    check(x, s, 4, 8)
    for dt in (torch.bfloat16, torch.float16):
        check((x * 1e-3).to(dt).clamp(-6e4, 6e4), s, 4, 8)


def test_beams_not_in_use_and_not_finite(cuda):
    x, s = rand_logits(cuda, 8, 3000, torch.bfloat16, 8)
    s[1] = s[2] = -math.inf
    s[4:6] = -math.inf
    x[1, 5] = math.nan  # not read
    check(x, s, 2, 4)
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    for row, place, value in ((0, 17, math.nan), (3, 2999, math.inf), (6, 0, -math.nan)):
        y = x.clone()
        y[row, place] = value
        with pytest.raises(ValueError, match="NaN"):
            paged.select_beams(y, s, 2, 4, check=True)
        err.zero_()
        got = paged.select_beams(y, s, 2, 4, check=False, err=err)
        assert int(err) == 256
        z = s.clone()
        z[row] = -math.inf  # what is left is as without this beam
        for a, b in zip(got, paged.select_beams(x, z, 2, 4)):
            assert torch.equal(a, b)
    for value in (math.nan, math.inf):
        z = s.clone()
        z[3] = value
        err.zero_()
        got = paged.select_beams(x, z, 2, 4, check=False, err=err)
        assert int(err) == 256 and 3 not in got.all_parents.tolist()[1]


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_nan_of_either_sign_in_every_wave(cuda, dtype):
    """Words of NaN lie above or below all others: the search for the best ends whatever they are."""
    V = 5000
    x, s = rand_logits(cuda, 6, V, DTYPES[dtype], 11)
    bits = x.view(torch.int32 if dtype == "fp32" else torch.int16)
    exp = {"bf16": 0x7f80, "fp16": 0x7c00, "fp32": 0x7f800000}[dtype]
    top = 0x7fffffff if dtype == "fp32" else 0x7fff
    signed = lambda v: v - 2 * (top + 1)  # with the sign
    bits[0, ::7], bits[1, ::7] = top, signed(exp + top + 1 + 1)
    bits[2, 100:164], bits[3, ::2] = signed(2 * top + 1), exp + 1
    bits[4, :] = signed(2 * top + 1)
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    for count in (3, 16, 17, 64):
        err.zero_()
        got = paged.select_beams(x, s, 3, count, check=False, err=err)
        assert int(err) == 256 and got.all_parents[0].tolist() == [-1] * count
        z = s.clone()
        z[:5] = -math.inf
        for a, b in zip(got, paged.select_beams(torch.where(torch.isnan(x), torch.zeros_like(x), x), z, 3, count)):
            assert torch.equal(a, b)


def test_scores_far_and_near(cuda):
    """Sums of log-probabilities far from zero, and beams a rounding apart."""
    x, s = rand_logits(cuda, 8, 4000, torch.float32, 9)
    s = torch.tensor([-1e6, -1e6 - 1, 0.0, -1e-30, -3e38, -3e38, 5.0, 5.0], device=cuda)
    check(x, s, 2, 16)
    # the same beam twice but for the last bit of one logit: order hangs on a sum's 1e-8
    y = x[:1].expand(4, -1).clone()
    y[1, 7] = torch.nextafter(y[1, 7], torch.tensor(10.0, device=cuda))
    check(y, torch.zeros(4, device=cuda), 4, 8)


def test_next_scores_over_the_scores_and_a_graph(cuda):
    x, s = rand_logits(cuda, 8, 6000, torch.bfloat16, 10)
    i32 = lambda *n: torch.full(n, -7, dtype=torch.int32, device=cuda)
    f32 = lambda *n: torch.full(n, -7.0, device=cuda)
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    live = s.clone()
    out = paged.BeamChoice(i32(8), i32(8), live, i32(2, 8), i32(2, 8), f32(2, 8))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        paged.select_beams(x, live, 4, 8, end_token=3, out=out, err=err, check=False)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged.select_beams(x, live, 4, 8, end_token=3, out=out, err=err)
    for seed in range(4):
        y, s = rand_logits(cuda, 8, 6000, torch.bfloat16, 20 + seed)
        x.copy_(y)
        live.copy_(s)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, paged.select_beams(y, s, 4, 8, end_token=3)):
            assert torch.equal(a, b)
    assert int(err) == 0


def test_no_requests(cuda):
    got = paged.select_beams(torch.empty((0, 10), device=cuda), torch.empty(0, device=cuda), 4)
    assert got.parents.shape == (0,) and got.all_tokens.shape == (0, 4)
