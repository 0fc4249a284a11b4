"""Products in 8-bit integers, attention over an encoder's states and over a paged cache, against their definitions in 64 bits.

Tolerances. A value rounded to a type is off by at most half a step, finfo.eps / 2 relative to it (`_half_step`).
* A product's sum is exact; it is turned into fp32, scaled twice and added to the bias in one more rounding: three half steps of
  fp32 of the scaled sum, one of the result's type.
* Attention: with a = sum_j p_j |v_j| / sum_j p_j, a relative error e of every p_j moves the result by at most 2 e a. e has the half step of
  P's type (tensor-core kernel; the other one keeps P in two parts and has the square of it), the error of a score and of
  exp2 (2^-20 covers exp2, the scaling of sums and the order of adding). A score's error is at most (size + 2) steps of fp32 of
  sum_d |q_d k_d| scale, the accumulator's additions being truncated. Then the result is rounded."""
import ctypes
import math
import threading

import numpy as np
import pytest
import torch

import dlf_b200
from dlf_b200 import gblas, gdnn, predict, tensor
from dlf_b200.gblas import BLASError, StatusCode

pytestmark = pytest.mark.gpu

TYPES = [torch.float16, torch.bfloat16, torch.float32]
HALF = [torch.float16, torch.bfloat16]


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _rand(seed, *shape):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed))


# ---------------------------------------------------------------------------------------------
# rows to 8-bit integers


def _quantized(x):
    """The definition: scales in fp32, quotients exact (53 bits tell a quotient of two 24-bit numbers from a tie)."""
    largest = x.double().abs().amax(1)
    scales = torch.clamp((largest / 127).float(), min=2.0 ** -126)
    q = torch.round(x.double() / scales.double().unsqueeze(1))
    bad = ~torch.isfinite(largest)
    scales[bad], q[bad] = math.nan, 0
    return q.to(torch.int8), scales


def _check_quantize(x, x_pad=(0, 0), q_pad=(0, 0)):
    rows, cols = x.shape
    wide = torch.full((rows, cols + sum(x_pad)), math.inf, dtype=x.dtype, device="cuda")  # (padding that would be seen)
    wide[:, x_pad[0]:x_pad[0] + cols] = x.cuda()
    out = torch.full((rows, cols + sum(q_pad)), 77, dtype=torch.int8, device="cuda")
    q, scales = tensor.quantize(wide[:, x_pad[0]:x_pad[0] + cols], out[:, q_pad[0]:q_pad[0] + cols])
    want_q, want_s = _quantized(x)
    assert torch.equal(scales.cpu().nan_to_num(-1), want_s.nan_to_num(-1))
    assert torch.equal(q.cpu(), want_q)
    assert bool((out[:, :q_pad[0]] == 77).all()) and bool((out[:, q_pad[0] + cols:] == 77).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (5, 8), (7, 33), (64, 129), (2500, 100), (2400, 300), (2400, 777), (2368, 2048),
                                       (17, 4096), (9, 11007), (5, 16391), (3, 40001)])
def test_quantize_sizes_and_alignments(dtype, rows, cols):
    x = (_rand(rows + cols, rows, cols) * torch.exp(_rand(cols, rows, 1))).clamp(-6e4, 6e4).to(dtype)
    _check_quantize(x)
    _check_quantize(x, (1, 2), (2, 3))
    _check_quantize(x, (3, 0), (5, 6))


@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_values_that_are_special(dtype):
    tiny, top = torch.finfo(dtype).tiny, torch.finfo(dtype).max
    rows = [[0.0] * 20, [-0.0] * 20, [math.inf] + [1.0] * 19, [1.0, -math.inf] + [2.0] * 18, [math.nan] + [1.0] * 19, [1.0] * 19 + [math.nan],
            [top] * 19 + [-top], [tiny] * 10 + [-tiny] * 10, [tiny / 4] * 20, [127.0] + [i + 0.5 for i in range(19)],
            [-127.0] + [-(i + 0.5) for i in range(19)], [12.7] + [0.05 * (2 * i + 1) for i in range(19)], [1.0] + [-1.0] * 19]
    _check_quantize(torch.tensor(rows, dtype=torch.float64).to(dtype))


def test_quantize_ties_and_their_neighbours():
    """Quotients at and one step beside the middle of two whole numbers, for scales that are and are not powers of two."""
    rows = []
    for scale in (1.0, 0.75, 1.0 / 3.0, 1.2345678, 3e-30, 7e30):
        s = np.float32(np.float32(127 * scale) / np.float32(127))
        mid = (np.arange(-126, 126) + 0.5).astype(np.float64) * float(s)
        x = mid.astype(np.float32)
        rows += [np.concatenate([[np.float32(127 * scale)], y]) for y in (x, np.nextafter(x, np.float32(np.inf)), np.nextafter(x, np.float32(-np.inf)))]
    _check_quantize(torch.from_numpy(np.stack(rows).astype(np.float32)))


def test_quantize_shapes_of_more_dimensions_and_allocation():
    x = _rand(3, 2, 5, 37).cuda().half()
    q, s = tensor.quantize(x)
    assert q.shape == x.shape and s.shape == (2, 5) and q.stride(1) % 16 == 0
    want_q, want_s = _quantized(x.cpu().view(10, 37))
    assert torch.equal(q.cpu().reshape(10, 37), want_q) and torch.equal(s.cpu().view(10), want_s)
    with pytest.raises(tensor.ShapeError):
        tensor.quantize(x.transpose(0, 1)[:, :, :])  # rows that no one stride leads through
    e = gblas.Event()
    buf, out, scales = x.view(-1), torch.empty(400, dtype=torch.int8, device="cuda"), torch.empty(10, device="cuda")
    gblas.quantizeRows(9, 37, buf, 37, 37, out, 3, 40, scales, event=e)
    assert torch.equal(out[3:363].view(9, 40)[:, :37].cpu(), want_q[1:]) and e.elapsed_ms() >= 0


# ---------------------------------------------------------------------------------------------
# products of 8-bit integers


def _check_product(m, n, k, dtype, bias=False, relu=False, seed=0, a_ld=0, b_ld=0, c_ld=0, a_off=0, b_off=0, extreme=False):
    g = torch.Generator().manual_seed(seed + m + 3 * n + 5 * k)
    a_ld, b_ld, c_ld = a_ld or k, b_ld or k, c_ld or n
    lo, hi = (-128, -127) if extreme else (-128, 128)
    a_all = torch.randint(lo, hi, (m * a_ld + a_off,), generator=g, dtype=torch.int8).cuda()
    b_all = torch.randint(lo, hi, (n * b_ld + b_off,), generator=g, dtype=torch.int8).cuda()
    a, b = a_all[a_off:].view(m, a_ld)[:, :k], b_all[b_off:].view(n, b_ld)[:, :k]
    sa = (torch.rand(m, generator=g) + 0.5).cuda()
    sb = ((torch.rand(n, generator=g) + 0.5) / (40 * math.sqrt(k) * (10 if extreme else 1))).cuda()
    bi = torch.randn(n, generator=g).to(dtype).cuda() if bias else None
    out = torch.full((m, c_ld), -7.0, dtype=dtype, device="cuda")
    y = tensor.matmul_int8(a, sa, b, sb, out[:, :n], bias=bi, activation="relu" if relu else None)
    scaled = (a.double() @ b.double().t()) * sb.double() * sa.double().unsqueeze(1)
    want = scaled + (bi.double() if bias else 0)
    if relu:
        want = want.clamp_min(0)
    tol = 3 * 2.0 ** -24 * (scaled.abs() + want.abs()) + _half_step(dtype) * want.abs() * (1 + 2.0 ** -20) + (2.0 ** -25 if dtype == torch.float16 else 0)
    worst = ((y.double() - want).abs() - tol).max().item()
    assert worst <= 0, worst
    assert bool((out[:, n:] == -7).all())
    assert dlf_b200.device_status() == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 128, 128), (2, 130, 40), (3, 5, 7), (16, 256, 512), (17, 300, 130), (33, 1000, 2048), (64, 64, 4096),
                                   (65, 200, 300), (128, 128, 128), (129, 257, 777), (256, 1000, 2048), (1111, 1537, 777), (300, 4096, 1024),
                                   (1500, 1500, 200), (2049, 1111, 333)])
def test_product_sizes(dtype, m, n, k):
    _check_product(m, n, k, dtype)
    _check_product(m, n, k, dtype, bias=True, relu=True, seed=1)


@pytest.mark.parametrize("m", [5, 100, 1300])
def test_product_strides_and_alignments(m):
    for kw in ({"a_ld": 320}, {"a_ld": 301, "b_ld": 303}, {"a_off": 16}, {"a_off": 5}, {"b_off": 3, "b_ld": 304}, {"c_ld": 1003}, {"c_ld": 1008},
               {"a_ld": 309, "b_ld": 333, "c_ld": 1001, "a_off": 1, "b_off": 2}):
        for dtype in (torch.float16, torch.float32):
            _check_product(m, 1000, 300, dtype, bias=True, **kw)


@pytest.mark.parametrize("m", [1, 70, 1100])
def test_product_of_the_greatest_depth_does_not_overflow(m):
    """131071 products of (-128) * (-128) are 2^31 - 16384."""
    _check_product(m, 3, 131071, torch.float32, extreme=True)


def test_product_scales_that_are_nan_or_infinite_reach_their_row_or_column_only():
    a, b = torch.ones(70, 32, dtype=torch.int8).cuda(), torch.ones(40, 32, dtype=torch.int8).cuda()
    sa, sb = torch.ones(70).cuda(), torch.ones(40).cuda()
    sa[3], sa[69], sb[5] = math.nan, math.inf, math.nan
    for m in (10, 70):
        for act in (None, "relu"):
            y = tensor.matmul_int8(a[:m], sa[:m], b, sb, activation=act).cpu()
            bad = torch.zeros(m, 40, dtype=torch.bool)
            bad[3], bad[:, 5] = True, True
            assert torch.equal(torch.isnan(y), bad)
            assert bool((y[~bad & ~torch.isinf(y)] == 32).all()) and int(torch.isinf(y).sum()) == (39 if m == 70 else 0)


def test_product_of_tensors_of_more_dimensions_and_events():
    a, b = torch.randint(-9, 9, (2, 3, 5, 48), dtype=torch.int8).cuda(), torch.randint(-9, 9, (7, 48), dtype=torch.int8).cuda()
    sa, sb = torch.rand(2, 3, 5).cuda(), torch.rand(7).cuda()
    e = gblas.Event()
    y = tensor.matmul_int8(a, sa, b, sb, dtype=torch.float32, event=e)
    want = (a.double() @ b.double().t()) * sa.double().unsqueeze(-1) * sb.double()
    assert y.shape == (2, 3, 5, 7) and torch.allclose(y.double(), want, rtol=4 * 2.0 ** -24, atol=0) and e.elapsed_ms() >= 0
    c = torch.zeros(100, device="cuda")
    gblas.gemmInt8(30, 3, 48, a.view(-1), 0, 48, sa.view(-1), b.view(-1), 48 * 2, 48, sb[2:5].contiguous(), c, 4, 3)
    assert torch.equal(c[4:94].view(30, 3), y.view(30, 7)[:, 2:5]) and float(c[:4].abs().sum()) == 0


def test_product_wait_that_runs_out_is_reported():
    """One tile whose last hand-over is left out (a test aid): the kernel gives up, returns and reports; the next call is sound."""
    a, b = torch.ones(8, 64, dtype=torch.int8).cuda(), torch.ones(8, 64, dtype=torch.int8).cuda()
    s = torch.ones(8).cuda()
    q = torch.zeros(1, 40, 1, 64, dtype=torch.float16, device="cuda")
    tensor.matmul_int8(a, s, b, s)
    gdnn.attention(q, q, q, torch.empty_like(q))
    assert dlf_b200.device_status() == 0
    L = dlf_b200.lib()
    try:
        L.dlf_b200_set_tuning(0, 0x10000000)
        tensor.matmul_int8(a, s, b, s)
        assert dlf_b200.device_status() & 1
        tensor.matmul_int8(a.repeat(10, 1), s.repeat(10), b, s)
        assert dlf_b200.device_status() & 1
        gdnn.attention(q, q, q, torch.empty_like(q))
        assert dlf_b200.device_status() & 1
    finally:
        L.dlf_b200_set_tuning(0, 0)
    assert bool((tensor.matmul_int8(a, s, b, s) == 64).all()) and dlf_b200.device_status() == 0


# ---------------------------------------------------------------------------------------------
# attention


def _attention_want(q, k, v, keep, scale):
    """The definition for one entry of the batch, in 64 bits, and the tolerance's parts: (y, a, score error) - q (queries, heads, size), k, v
    (keys, kv_heads, size), keep (keys)."""
    lq, h, d = q.shape
    group = h // k.shape[1]
    y, a = torch.zeros(q.shape, dtype=torch.float64, device=q.device), torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    e = torch.zeros(lq, h, 1, dtype=torch.float64, device=q.device)
    at = keep.nonzero().view(-1)
    if len(at):
        for x in range(h):
            kk, vv, qq = k[at, x // group].double(), v[at, x // group].double(), q[:, x].double()
            p = torch.softmax(qq @ kk.t() * scale, -1)
            y[:, x], a[:, x] = p @ vv, p @ vv.abs()
            e[:, x] = ((qq.abs() @ kk.abs().t()).amax(1, keepdim=True) * scale * (d + 2) * 2.0 ** -23)
    return y, a, e


def _check_rows(y, want, a, e, dtype, p_error):
    assert torch.isfinite(y.float()).all()
    tol = 2 * (p_error + e + 2.0 ** -20) * a + _half_step(dtype) * (want.abs() + 2 * (p_error + e) * a) + (2.0 ** -25 if dtype == torch.float16 else 0)
    worst = ((y.double() - want).abs() - tol).max().item()
    assert worst <= 0, worst


def _check_attention(b, lq, lk, h, hk, d, dtype, padding="none", garbage=True, seed=0, scale=None, spread=1.0, layout="packed", shared=False):
    g = torch.Generator(device="cuda").manual_seed(seed + 7 * b + 11 * lq + 13 * lk + d)

    def rand(*shape):
        return (torch.randn(shape, generator=g, device="cuda") * spread).to(dtype)

    kb = 1 if shared else b
    if layout == "packed":  # keys and values of one projection
        q, (k, v) = rand(1 if shared else b, lq, h, d).expand(b, -1, -1, -1), rand(kb, lk, 2, hk, d).unbind(2)
        y = torch.full((b, lq, h, d), 7.0, dtype=dtype, device="cuda")
    else:  # heads before tokens, lines with room behind them
        q, k, v = (rand(x, n, m, d + 8)[..., :d].transpose(1, 2) for x, n, m in ((b, h, lq), (kb, hk, lk), (kb, hk, lk)))
        y = torch.full((b, h, lq, d + 24), 7.0, dtype=dtype, device="cuda")[..., :d].transpose(1, 2)
    keep = torch.ones(b, lk, dtype=torch.bool, device="cuda")
    lengths = mask = None
    if padding in ("lengths", "both"):
        lengths = torch.randint(0, lk + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
        lengths[0] = lk
        if b > 1:
            lengths[b - 1] = 0
        keep &= torch.arange(lk, device="cuda") < lengths.unsqueeze(1)
    if padding == "one mask":
        mask = (torch.rand(1, lk, generator=g, device="cuda") < 0.6).expand(b, -1)
        keep &= mask
    if padding in ("mask", "both"):
        mask = torch.rand(b, lk, generator=g, device="cuda") < 0.6
        if b > 1:
            mask[1] = False
        keep &= mask
    if garbage and not shared:
        k[~keep], v[~keep] = math.nan, math.inf
    kx, vx = (k.expand(b, -1, -1, -1), v.expand(b, -1, -1, -1)) if shared else (k, v)
    gdnn.attention(q, kx, vx, y, scale=scale, key_lengths=lengths, key_mask=mask)
    few = lq <= (8 if lk <= 128 else 32 if d <= 64 else 16)  # the kernel that keeps P in two parts; the others round it once, half a step each
    for i in range(b):
        want, a, e = _attention_want(q[i], kx[i], vx[i], keep[i], scale or 1 / math.sqrt(d))
        _check_rows(y[i], want, a, e, dtype, _half_step(dtype) ** 2 if few else _half_step(dtype))
        if not keep[i].any():
            assert float(y[i].float().abs().sum()) == 0
    assert dlf_b200.device_status() == 0


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("padding", ["none", "lengths", "mask", "both"])
@pytest.mark.parametrize("lq,lk,h,hk", [(1, 1, 1, 1), (1, 15, 2, 1), (1, 65, 16, 2), (1, 200, 32, 2), (2, 777, 16, 2), (4, 129, 4, 4), (1, 3000, 8, 8)])
@pytest.mark.parametrize("d", [64, 128])
def test_attention_of_few_queries(dtype, padding, lq, lk, h, hk, d):
    _check_attention(3, lq, lk, h, hk, d, dtype, padding)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("padding", ["none", "lengths", "mask", "both"])
@pytest.mark.parametrize("lq,lk,h,hk", [(17, 1, 1, 1), (32, 16, 4, 2), (100, 77, 8, 8), (128, 128, 2, 1), (129, 127, 3, 3), (257, 129, 4, 1), (300, 640, 4, 2),
                                        (5, 1000, 8, 1)])
@pytest.mark.parametrize("d", [64, 128])
def test_attention_of_many_queries(dtype, padding, lq, lk, h, hk, d):
    _check_attention(3, lq, lk, h, hk, d, dtype, padding)


@pytest.mark.parametrize("d", [40, 64, 96, 128])
@pytest.mark.parametrize("lk", [1, 16, 17, 64, 77, 80, 81, 96, 97, 112, 128])
def test_attention_of_many_queries_over_few_keys(d, lk):
    """One tile of keys: sizes on either side of its steps, entries without keys between others."""
    for i, padding in enumerate(("none", "lengths", "mask", "both")):
        _check_attention(3, (8, 9, 20, 32)[i], lk, 4, 1, d, HALF[i % 2], padding, seed=lk)
        _check_attention(4, 33 + 50 * i, lk, 4, 2, d, HALF[i % 2], padding, seed=lk)
        _check_attention(3, 150, lk, 3, 1, d, HALF[1 - i % 2], padding, layout="heads first")


@pytest.mark.parametrize("d", [64, 80, 128])
@pytest.mark.parametrize("lk", [60, 120])
def test_attention_over_few_keys_that_the_batch_shares(d, lk):
    _check_attention(5, 140, lk, 4, 2, d, torch.float16, "lengths", shared=True)
    _check_attention(5, 140, lk, 4, 4, d, torch.bfloat16, "one mask", shared=True)


@pytest.mark.parametrize("d,lk", [(64, 77), (64, 128), (128, 50), (128, 128)])
def test_attention_over_few_keys_with_many_tiles_a_block(d, lk):
    """More tiles of queries than blocks, so that a block goes on to other queries, heads and entries, some of them without keys."""
    _check_attention(9, 600, lk, 24, 8, d, torch.bfloat16, "lengths")
    _check_attention(6, 700, lk, 20, 20, d, torch.float16, "both")


def test_attention_wait_that_runs_out_is_reported_over_many_keys():
    q, k = (torch.ones(1, n, 1, 64, dtype=torch.float16, device="cuda") for n in (200, 250))
    y = torch.empty_like(q)
    gdnn.attention(q, k, k, y)
    L = dlf_b200.lib()
    try:
        L.dlf_b200_set_tuning(0, 0x10000000)
        gdnn.attention(q, k, k, torch.empty_like(q))
        assert dlf_b200.device_status() & 1
    finally:
        L.dlf_b200_set_tuning(0, 0)
    y = torch.empty_like(q)
    gdnn.attention(q, k, k, y)
    assert bool((y == 1).all()) and dlf_b200.device_status() == 0


@pytest.mark.parametrize("d", [8, 16, 40, 72, 80, 96, 120])
@pytest.mark.parametrize("lq", [1, 40])
def test_attention_head_sizes(d, lq):
    for padding in ("none", "lengths", "mask"):
        _check_attention(2, lq, 150, 4, 2, d, torch.float16, padding)


@pytest.mark.parametrize("lq", [1, 3, 150])
@pytest.mark.parametrize("d", [64, 80, 128])
def test_attention_layouts_and_shared_states(lq, d):
    _check_attention(3, lq, 190, 4, 2, d, torch.bfloat16, "lengths", layout="heads first")
    _check_attention(3, lq, 190, 4, 2, d, torch.bfloat16, "mask", layout="heads first")
    _check_attention(3, lq, 190, 4, 2, d, torch.float16, "lengths", shared=True)
    _check_attention(3, lq, 190, 4, 2, d, torch.float16, "one mask", shared=True)
    _check_attention(1, lq, 190, 4, 1, d, torch.float16, layout="heads first")


@pytest.mark.parametrize("lq", [1, 200])
@pytest.mark.parametrize("d", [64, 128])
def test_attention_scores_that_grow_and_scales(lq, d):
    """Scores of up to some hundreds, keys in rising order, so that the reference maximum moves time and again."""
    for dtype in HALF:
        _check_attention(2, lq, 700, 2, 2, d, dtype, spread=4.0, scale=0.3, seed=1)
        q = torch.ones(1, lq, 2, d, dtype=dtype, device="cuda")
        k = (torch.arange(700, device="cuda") * 0.05).to(dtype).view(1, 700, 1, 1).expand(1, 700, 2, d).contiguous()
        v = torch.randn(1, 700, 2, d, device="cuda").to(dtype)
        for order in (k, k.flip(1), -k):
            y = torch.empty_like(q)
            gdnn.attention(q, order, v, y, scale=0.5)
            want, a, e = _attention_want(q[0], order[0], v[0], torch.ones(700, dtype=torch.bool, device="cuda"), 0.5)
            _check_rows(y[0], want, a, e, dtype, _half_step(dtype) if lq > 32 else _half_step(dtype) ** 2)


@pytest.mark.parametrize("scale", [1.7e-38, 1e-38, 1e-44])
def test_attention_scales_that_leave_nothing_between_the_keys(scale):
    """The mean of the kept values, whichever kernel takes the call."""
    for dtype in HALF:
        for lq, lk in ((1, 300), (1, 3000), (20, 300), (200, 300), (200, 100)):
            _check_attention(2, lq, lk, 4, 2, 64, dtype, "lengths", scale=scale)
        g = torch.Generator(device="cuda").manual_seed(1)
        table, kp, vp = _cache(g, 2, 100, 16, 2, 64, dtype)
        q = torch.randn(2, 4, 64, generator=g, device="cuda").to(dtype)
        y = torch.empty_like(q)
        gdnn.paged_attention(q, kp, vp, table, torch.tensor([100, 33], dtype=torch.int32, device="cuda"), y, scale=scale)
        for i, n in enumerate((100, 33)):
            k, v = (t[table[i].long()].reshape(-1, 2, 64)[:n] for t in (kp, vp))
            want, a, e = _attention_want(q[i:i + 1], k, v, torch.ones(n, dtype=torch.bool, device="cuda"), scale)
            _check_rows(y[i:i + 1], want, a, e, dtype, _half_step(dtype) ** 2)


@pytest.mark.parametrize("lq,lk", [(1, 300), (20, 300), (200, 300), (200, 100), (1, 60000), (40, 9000)])
@pytest.mark.parametrize("d", [64, 128])
def test_attention_scores_beyond_the_range_of_exp2(lq, lk, d):
    """Scores whose distance, and whose own rounding once they are scaled, is more than exp2 can take: what counts are the keys with
    the greatest score, equally. The scores are exact in fp32 (whole numbers below 2^8 times a power of two), so no error of theirs is left."""
    g = torch.Generator(device="cuda").manual_seed(lk + d)
    at = torch.randint(1, 200, (1, lk, 2, 1), generator=g, device="cuda")
    for dtype, q_size, k_size, scale in ((torch.float16, 2.0 ** 15, 2.0 ** 8, None), (torch.bfloat16, 2.0 ** 15, 2.0 ** 8, None), (torch.bfloat16, 2.0 ** 40, 2.0 ** 30, None),
                                         (torch.float16, 1.0, 1.0, 1e30), (torch.bfloat16, 1.0, 1.0, 1e35), (torch.float16, 2.0 ** 15, 2.0 ** 8, 1e20)):
        q = torch.full((1, lq, 4, d), q_size, device="cuda").to(dtype)
        q[:, 1::2], q[:, :, 1] = -q[:, 1::2], -q[:, :, 1]
        k = (at * k_size).expand(-1, -1, -1, d).to(dtype).contiguous()
        v = torch.randn(1, lk, 2, d, generator=g, device="cuda").to(dtype)
        y = torch.full_like(q, 7)
        gdnn.attention(q, k, v, y, scale=scale)
        want, a, e = _attention_want(q[0], k[0], v[0], torch.ones(lk, dtype=torch.bool, device="cuda"), scale or 1 / math.sqrt(d))
        _check_rows(y[0], want, a, 0 * e, dtype, _half_step(dtype))
    table, kp, vp = _cache(g, 1, 400, 16, 2, d, torch.float16)
    kp.copy_((torch.randint(1, 200, kp.shape[:3] + (1,), generator=g, device="cuda") * 2.0 ** 8).expand(-1, -1, -1, d))
    q = torch.full((1, 4, d), 2.0 ** 15, dtype=torch.float16, device="cuda")
    y = torch.full_like(q, 7)
    gdnn.paged_attention(q, kp, vp, table, torch.tensor([400], dtype=torch.int32, device="cuda"), y)
    k, v = (t[table[0].long()].reshape(-1, 2, d) for t in (kp, vp))
    want, a, e = _attention_want(q, k, v, torch.ones(400, dtype=torch.bool, device="cuda"), 1 / math.sqrt(d))
    _check_rows(y, want, a, 0 * e, torch.float16, _half_step(torch.float16) ** 2)


@pytest.mark.parametrize("b,lq,lk", [(1000, 1, 4096), (400, 20, 4096), (200, 64, 4096), (2, 200, 40000), (3, 200, 128), (3, 200, 60)])
@pytest.mark.parametrize("d", [64, 128])
def test_attention_of_many_keys_that_one_outweighs(b, lq, lk, d):
    """One key is e^17.5 times as heavy as every other and has zeros for values: what is read is the others' sum. In fp16 a p below 2^-14
    has fewer bits, a step of 2^-24: with p times 2^7 that is an error of 2^-32 of the heaviest for every key (over few keys times
    2^15 and less than that)."""
    for dtype in HALF:
        for heavy in (0, lk // 3):
            q, k, v = torch.zeros(1, 1, 1, d), torch.zeros(1, lk, 1, d), torch.ones(1, lk, 1, d)
            q[..., 0], k[:, heavy, :, 0], v[:, heavy] = 1, 17.5, 0
            q, k, v = (t.to(dtype).cuda() for t in (q, k, v))
            y = torch.full((b, lq, 1, d), 7.0, dtype=dtype, device="cuda")
            gdnn.attention(q.expand(b, lq, -1, -1).contiguous(), k.expand(b, -1, -1, -1), v.expand(b, -1, -1, -1), y, scale=1.0)
            want, a, e = _attention_want(q[0], k[0], v[0], torch.ones(lk, dtype=torch.bool, device="cuda"), 1.0)
            lost = lk * 2.0 ** -32 if dtype == torch.float16 else 0.0
            want, a = (t.expand(b, lq, -1, -1) for t in (want, a + lost / 2 / _half_step(dtype)))  # (so that 2 half steps of a hold it)
            _check_rows(y, want, a, e, dtype, _half_step(dtype))


@pytest.mark.parametrize("b,lq,lk,h,hk,d", [(1, 256, 40000, 1, 1, 64), (1, 40, 9000, 2, 1, 128), (2, 300, 5000, 3, 1, 80), (1, 1, 60000, 4, 1, 128)])
def test_attention_over_many_keys_is_cut_and_joined(b, lq, lk, h, hk, d):
    _check_attention(b, lq, lk, h, hk, d, torch.bfloat16, "lengths")
    _check_attention(b, lq, lk, h, hk, d, torch.float16, "mask", seed=1)


@pytest.mark.parametrize("lq", [1, 60])
@pytest.mark.parametrize("lk", [100, 1000])
def test_attention_infinities_and_nan_that_count_reach_their_rows_only(lq, lk):
    """A NaN or infinite score makes its row NaN (inf - inf), whichever CTA meets it; other rows, heads and entries do not see it."""
    q = torch.randn(2, lq, 2, 64, device="cuda").half()
    k, v = torch.randn(2, lk, 2, 64, device="cuda").half(), torch.randn(2, lk, 2, 64, device="cuda").half()
    good = torch.empty_like(q)
    gdnn.attention(q, k, v, good)
    for value in (math.nan, math.inf):
        kx = k.clone()
        kx[1, lk - 2, 1] = value
        y = torch.empty_like(q)
        gdnn.attention(q.abs(), kx, v, y)  # (positive queries: the score is +infinity)
        clean = torch.empty_like(q)
        gdnn.attention(q.abs(), k, v, clean)
        assert torch.isnan(y[1, :, 1]).all()
        assert torch.equal(y[0], clean[0]) and torch.equal(y[1, :, 0], clean[1, :, 0])
    qx = q.clone()
    qx[0, lq - 1, 0, 3] = math.nan
    y = torch.empty_like(q)
    gdnn.attention(qx, k, v, y)
    assert torch.isnan(y[0, lq - 1, 0]).all()
    y[0, lq - 1, 0] = good[0, lq - 1, 0]
    assert torch.equal(y, good)


def test_attention_lengths_that_do_not_fit_are_cut_and_reported():
    for lq in (1, 50):
        q, k = torch.randn(3, lq, 2, 64, device="cuda").half(), torch.randn(3, 90, 2, 64, device="cuda").half()
        want, y = torch.empty_like(q), torch.empty_like(q)
        gdnn.attention(q, k, k, want, key_lengths=torch.tensor([90, 0, 5], dtype=torch.int32, device="cuda"))
        assert dlf_b200.device_status() == 0
        gdnn.attention(q, k, k, y, key_lengths=torch.tensor([1 << 30, -4, 5], dtype=torch.int32, device="cuda"))
        assert dlf_b200.device_status() == 2
        assert torch.equal(y, want)


def test_attention_refusals_on_the_device():
    def refused(code, *args, **kw):
        with pytest.raises(BLASError) as e:
            gdnn.attention(*args, **kw)
        assert e.value.status == code

    q, k = torch.zeros(2, 20, 4, 64, dtype=torch.float16, device="cuda"), torch.zeros(2, 30, 2, 64, dtype=torch.float16, device="cuda")
    y = torch.empty_like(q)
    refused(StatusCode.kInvalidMatrixA, q.cpu(), k, k, y)
    refused(StatusCode.kInvalidMatrixA, q, k, k, y, key_lengths=torch.zeros(2, dtype=torch.int32))
    refused(StatusCode.kInvalidValue, q, k, k, y, key_lengths=torch.zeros(2, dtype=torch.int64, device="cuda"))
    refused(StatusCode.kInvalidDimension, q, k, k, y, key_lengths=torch.zeros(3, dtype=torch.int32, device="cuda"))
    refused(StatusCode.kInvalidValue, q, k, k, y, key_mask=torch.zeros(2, 30, device="cuda"))
    refused(StatusCode.kInvalidValue, q, k, k, y, key_mask=torch.zeros(2, 29, dtype=torch.bool, device="cuda"))
    refused(StatusCode.kInvalidValue, q, k, k, y, key_mask=torch.zeros(30, 2, dtype=torch.bool, device="cuda").t())
    refused(StatusCode.kInvalidDimension, q, k, k[:, :29], y)
    refused(StatusCode.kInvalidDimension, q, k[:1], k[:1], y)
    refused(StatusCode.kInvalidDimension, q[:, :0], k, k, y[:, :0])
    refused(StatusCode.kInvalidDimension, q, k[:, :0], k[:, :0], y)
    refused(StatusCode.kInvalidDimension, q[:, :, :3], k, k, y[:, :, :3])
    refused(StatusCode.kInvalidValue, q, k, k, y, scale=0.0)
    refused(StatusCode.kNotImplemented, q.float(), k.float(), k.float(), y.float())
    refused(StatusCode.kNotImplemented, q[..., 1:57], k[..., :56], k[..., :56], y[..., :56])  # starts off a 16-byte boundary
    refused(StatusCode.kNotImplemented, q[..., :60], k[..., :60], k[..., :60], y[..., :60])
    refused(StatusCode.kInvalidLeadDimC, q, k, k, y[:1].expand(2, -1, -1, -1))
    wide = torch.zeros(2, 30, 2, 68, dtype=torch.float16, device="cuda")[..., :64]  # strides that are no multiple of 8
    refused(StatusCode.kNotImplemented, q, wide, wide, y)


# ---------------------------------------------------------------------------------------------
# the paged cache


def _cache(g, b, longest, page, hk, d, dtype, layout="pages"):
    per = -(-longest // page)
    pages = b * per + 3
    table = torch.randperm(pages, generator=g, device="cuda")[:b * per].to(torch.int32).view(b, per)
    shape = (pages, page, hk, d)
    if layout == "pages":
        kp, vp = (torch.randn(shape, generator=g, device="cuda").to(dtype) for _ in range(2))
    else:  # keys and values of a page together, heads before tokens
        both = torch.randn((pages, 2, hk, page, d), generator=g, device="cuda").to(dtype)
        kp, vp = both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)
    return table, kp, vp


def _check_paged(b, longest, page, h, hk, d, dtype, layout="pages", seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + b + 3 * longest + 5 * page + d)
    table, kp, vp = _cache(g, b, longest, page, hk, d, dtype, layout)
    lengths = torch.randint(0, longest + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
    lengths[0] = longest
    if b > 1:
        lengths[1] = 0
    pos = torch.arange(table.shape[1] * page, device="cuda")
    flat = table.long()[:, pos // page] * page + pos % page
    keep = pos < lengths.unsqueeze(1)
    unused = torch.ones(kp.shape[:2], dtype=torch.bool, device="cuda").view(-1)
    unused[flat[keep]] = False
    kp[unused.view(kp.shape[:2])], vp[unused.view(kp.shape[:2])] = math.nan, math.inf  # whatever is left in freed places
    # table entries behind a sequence's length may be anything
    beyond = torch.arange(table.shape[1], device="cuda") * page >= lengths.unsqueeze(1)
    table = torch.where(beyond, torch.full_like(table, -1), table)
    q = torch.randn((b, h, d), generator=g, device="cuda").to(dtype)
    y = torch.full_like(q, 7.0)
    gdnn.paged_attention(q, kp, vp, table, lengths, y)
    k, v = (t.reshape(-1, hk, d) for t in (kp, vp))
    for i in range(b):
        n = int(lengths[i])
        at = flat[i, :n]
        want, a, e = _attention_want(q[i:i + 1], k[at], v[at], torch.ones(n, dtype=torch.bool, device="cuda"), 1 / math.sqrt(d))
        _check_rows(y[i:i + 1], want, a, e, dtype, _half_step(dtype) ** 2)
    assert float(y[1 if b > 1 else 0].float().abs().sum()) == 0 or b == 1
    assert dlf_b200.device_status() == 0


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("d", [64, 80, 128])
@pytest.mark.parametrize("b,longest,page,h,hk", [(1, 1, 1, 1, 1), (4, 130, 16, 4, 4), (7, 300, 24, 8, 2), (3, 1000, 8, 32, 1), (40, 500, 128, 8, 4), (2, 5000, 16, 20, 1),
                                                 (3, 100, 1, 2, 2), (2, 700, 48, 9, 1), (2, 20000, 64, 4, 2)])
def test_paged_attention(dtype, d, b, longest, page, h, hk):
    _check_paged(b, longest, page, h, hk, d, dtype)


@pytest.mark.parametrize("page", [5, 16])
def test_paged_attention_other_layouts(page):
    _check_paged(3, 200, page, 8, 2, 64, torch.float16, layout="heads first")
    _check_paged(3, 200, page, 8, 2, 128, torch.bfloat16, layout="heads first")


def test_paged_attention_many_sequences():
    _check_paged(300, 90, 16, 2, 1, 64, torch.bfloat16)


@pytest.mark.parametrize("b,longest,hk", [(3000, 40, 2), (1200, 700, 1), (20000, 64, 4), (5000, 65, 1)])
def test_paged_attention_thousands_of_sequences(b, longest, hk):
    """Sequences that a CTA has whole, and those that its end cuts, each once, empty ones among them."""
    g = torch.Generator(device="cuda").manual_seed(b)
    table, kp, vp = _cache(g, b, longest, 16, hk, 64, torch.float16)
    lengths = torch.randint(0, longest + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
    q = torch.randn((b, 4, 64), generator=g, device="cuda").half()
    y = torch.full_like(q, 7.0)
    gdnn.paged_attention(q, kp, vp, table, lengths, y)
    for i in range(0, b, 1000):
        k, v = (t[table[i:i + 1000].long()].flatten(1, 2).double().repeat_interleave(4 // hk, 2) for t in (kp, vp))
        keep = torch.arange(k.shape[1], device="cuda") < lengths[i:i + 1000, None]
        s = (torch.einsum("bhd,bkhd->bhk", q[i:i + 1000].double(), k) / 8).masked_fill(~keep[:, None], -math.inf)
        p = torch.softmax(s, -1).nan_to_num(0.0)
        want, a = torch.einsum("bhk,bkhd->bhd", p, v), torch.einsum("bhk,bkhd->bhd", p, v.abs())
        e = torch.einsum("bhd,bkhd->bhk", q[i:i + 1000].double().abs(), k.abs()).amax(-1, keepdim=True) / 8 * 66 * 2.0 ** -23
        _check_rows(y[i:i + 1000], want, a, e, torch.float16, _half_step(torch.float16) ** 2)
    assert dlf_b200.device_status() == 0


@pytest.mark.parametrize("page", [6, 16])
def test_pages_and_lengths_that_do_not_exist_are_left_out_and_reported(page):
    g = torch.Generator(device="cuda").manual_seed(page)
    table, kp, vp = _cache(g, 3, 10 * page, page, 2, 64, torch.float16)
    lengths = torch.tensor([10 * page, 9 * page + 1, 5], dtype=torch.int32, device="cuda")
    q = torch.randn(3, 4, 64, generator=g, device="cuda").half()
    y = torch.empty_like(q)
    bad = table.clone()
    bad[0, 4], bad[1, 0] = kp.shape[0], -1
    gdnn.paged_attention(q, kp, vp, bad, lengths, y)
    assert dlf_b200.device_status() == 2
    pos = torch.arange(10 * page, device="cuda")
    for i in range(3):
        keep = (pos < lengths[i]) & (bad[i].long()[pos // page] >= 0) & (bad[i].long()[pos // page] < kp.shape[0])
        at = (table[i].long()[pos // page] * page + pos % page)
        k, v = (t.reshape(-1, 2, 64)[at] for t in (kp, vp))
        want, a, e = _attention_want(q[i:i + 1], k, v, keep, 1 / 8)
        _check_rows(y[i:i + 1], want, a, e, torch.float16, _half_step(torch.float16) ** 2)
    want = torch.empty_like(q)
    gdnn.paged_attention(q, kp, vp, table, torch.tensor([10 * page, 0, 5], dtype=torch.int32, device="cuda"), want)
    assert dlf_b200.device_status() == 0
    gdnn.paged_attention(q, kp, vp, table, torch.tensor([2000000000, -7, 5], dtype=torch.int32, device="cuda"), y)
    assert dlf_b200.device_status() == 2 and torch.equal(y, want)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("layout", ["pages", "heads first"])
@pytest.mark.parametrize("page,hk,d", [(16, 8, 128), (7, 3, 40)])
def test_paged_append(dtype, layout, page, hk, d):
    g = torch.Generator(device="cuda").manual_seed(5)
    table, kp, vp = _cache(g, 4, 100, page, hk, d, dtype, layout)
    want_k, want_v = kp.clone(), vp.clone()
    tokens = torch.randn(2, 60, 2, hk, d, generator=g, device="cuda").to(dtype)  # (keys and values beside each other)
    k, v = tokens[0].unbind(1)
    pos = torch.cat([torch.arange(50, device="cuda"), torch.tensor([99, 0, 50, 98, 3, 4, 5, 6, 7, 8], device="cuda")]).to(torch.int32)
    seq = torch.cat([torch.full((50,), 2, device="cuda"), torch.tensor([0, 0, 0, 1, 3, 3, 3, 3, 3, 3], device="cuda")]).to(torch.int32)
    gdnn.paged_append(k, v, kp, vp, table, pos, seq)
    at = table.long()[seq.long(), pos.long() // page]
    want_k[at, pos.long() % page], want_v[at, pos.long() % page] = k, v
    assert torch.equal(kp, want_k) and torch.equal(vp, want_v)
    # without sequences: the i-th token is the i-th sequence's; fewer tokens than sequences
    k, v = tokens[1, :3].unbind(1)
    pos = torch.tensor([7, 99, 0], dtype=torch.int32, device="cuda")
    gdnn.paged_append(k, v, kp, vp, table, pos)
    at = table.long()[torch.arange(3, device="cuda"), pos.long() // page]
    want_k[at, pos.long() % page], want_v[at, pos.long() % page] = k, v
    assert torch.equal(kp, want_k) and torch.equal(vp, want_v) and dlf_b200.device_status() == 0


def test_paged_append_leaves_out_what_does_not_exist():
    g = torch.Generator(device="cuda").manual_seed(6)
    table, kp, vp = _cache(g, 2, 40, 10, 2, 64, torch.float16)
    table[1, 2] = kp.shape[0]
    k = torch.randn(7, 2, 64, generator=g, device="cuda").half()
    before_k, before_v = kp.clone(), vp.clone()
    pos = torch.tensor([-1, 40, 5, 5, 25, 2147483647, 3], dtype=torch.int32, device="cuda")
    seq = torch.tensor([0, 0, -1, 2, 1, 0, 1], dtype=torch.int32, device="cuda")
    gdnn.paged_append(k, k, kp, vp, table, pos, seq)
    assert dlf_b200.device_status() == 2
    before_k[table[1, 0].long(), 3], before_v[table[1, 0].long(), 3] = k[6], k[6]  # the only one with a place
    assert torch.equal(kp, before_k) and torch.equal(vp, before_v)


def test_a_padded_batch_appends_and_attends_without_a_report():
    """Sequences of length 0 (positions -1) between others, their table entries anything."""
    g = torch.Generator(device="cuda").manual_seed(8)
    table, kp, vp = _cache(g, 5, 40, 10, 2, 64, torch.float16)
    n = torch.tensor([0, 17, 0, 40, -1], dtype=torch.int32, device="cuda")
    table[n <= 0] = 2 ** 31 - 1
    q, k = (torch.randn(5, h, 64, generator=g, device="cuda").half() for h in (4, 2))
    want_k = kp.clone()
    for i in (1, 3):
        last = int(n[i]) - 1
        want_k[table[i, last // 10].long(), last % 10] = k[i]
    gdnn.paged_append(k, k, kp, vp, table, n - 1)
    y = torch.full_like(q, float("nan"))
    gdnn.paged_attention(q, kp, vp, table, n, y)
    assert dlf_b200.device_status() == 0
    assert torch.equal(kp, want_k)
    for i in range(5):
        if n[i] <= 0:
            assert bool((y[i] == 0).all())
        else:
            flat = kp[table[i].long()].reshape(-1, 2, 64)[:n[i]], vp[table[i].long()].reshape(-1, 2, 64)[:n[i]]
            want, a, e = _attention_want(q[i:i + 1], *flat, torch.ones(int(n[i]), dtype=torch.bool, device="cuda"), 1 / 8)
            _check_rows(y[i:i + 1], want, a, e, torch.float16, _half_step(torch.float16) ** 2)


def test_paged_append_the_same_place_twice_holds_one_of_the_two_in_every_piece():
    table, kp, vp = _cache(torch.Generator(device="cuda").manual_seed(7), 1, 16, 16, 1, 64, torch.float16)
    k = torch.stack([torch.full((1, 64), 1.0), torch.full((1, 64), 2.0)]).cuda().half()
    where = torch.zeros(2, dtype=torch.int32, device="cuda")
    gdnn.paged_append(k, -k, kp, vp, table, where, where)
    got = kp[table[0, 0].long(), 0]
    assert bool(((got == 1) | (got == 2)).all())


def test_paged_refusals_on_the_device():
    table, kp, vp = _cache(torch.Generator(device="cuda").manual_seed(8), 2, 40, 10, 2, 64, torch.float16)
    q, n = torch.zeros(2, 4, 64, dtype=torch.float16, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    y = torch.empty_like(q)

    def refused(code, *args):
        with pytest.raises(BLASError) as e:
            gdnn.paged_attention(*args)
        assert e.value.status == code

    refused(StatusCode.kInvalidValue, q, kp, vp, table.long(), n, y)
    refused(StatusCode.kInvalidValue, q, kp, vp.bfloat16(), table, n, y)
    refused(StatusCode.kInvalidDimension, q, kp, vp[:-1], table, n, y)
    refused(StatusCode.kInvalidDimension, q, kp, vp, table[:1], n, y)
    refused(StatusCode.kInvalidDimension, q, kp, vp, table, n[:1], y)
    refused(StatusCode.kInvalidDimension, q[:, :3], kp, vp, table, n, y[:, :3])
    refused(StatusCode.kInvalidMatrixA, q, kp, vp, table.cpu(), n, y)
    refused(StatusCode.kNotImplemented, q.float(), kp.float(), vp.float(), table, n, y.float())
    with pytest.raises(BLASError) as e:
        gdnn.paged_append(kp[0, :2], vp[0, :2], kp[:1].expand(4, -1, -1, -1), vp[:4], table, n)
    assert e.value.status == StatusCode.kInvalidLeadDimC  # pages that are one
    with pytest.raises(BLASError) as e:
        gdnn.paged_append(kp[0], vp[0], kp, vp, table, torch.zeros(10, dtype=torch.int32, device="cuda"))
    assert e.value.status == StatusCode.kInvalidDimension  # more tokens than sequences


# ---------------------------------------------------------------------------------------------
# streams, threads, graphs, scratch


def _calls(seed):
    """One call of each operator that uses scratch, as (function of a queue that makes it, its output, what it is to be)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    a, b = (torch.randint(-99, 99, (n, 333), generator=g, device="cuda", dtype=torch.int8) for n in (200, 150))  # odd lines: copied first
    sa, sb = torch.rand(200, generator=g, device="cuda"), torch.rand(150, generator=g, device="cuda")
    c = torch.empty(200, 150, device="cuda")
    q, k = torch.randn(2, 1, 8, 64, generator=g, device="cuda").half(), torch.randn(2, 4000, 2, 64, generator=g, device="cuda").half()
    y = torch.empty_like(q)
    q2, y2 = (torch.randn(1, 200, 2, 128, generator=g, device="cuda").bfloat16() for _ in range(2))
    k2 = torch.randn(1, 3000, 1, 128, generator=g, device="cuda").bfloat16()
    table, kp, vp = _cache(g, 3, 2000, 16, 2, 64, torch.float16)
    n = torch.tensor([2000, 17, 900], dtype=torch.int32, device="cuda")
    q3 = torch.randn(3, 4, 64, generator=g, device="cuda").half()
    y3 = torch.empty_like(q3)
    calls = [(lambda s: tensor.matmul_int8(a, sa, b, sb, c, queue=s), c), (lambda s: gdnn.attention(q, k, k, y, queue=s), y),
             (lambda s: gdnn.attention(q2, k2, k2, y2, queue=s), y2), (lambda s: gdnn.paged_attention(q3, kp, vp, table, n, y3, queue=s), y3)]
    done = []
    for f, out in calls:
        f(None)
        done.append((f, out, out.clone()))
    return done


def test_operators_on_another_stream_and_from_several_threads():
    calls = _calls(1)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for f, out, want in calls:
        out.zero_()
        side.wait_stream(torch.cuda.current_stream())
        f(side)
        side.synchronize()
        assert torch.equal(out, want)
    errors = []

    def work(i, stream):
        try:
            mine = _calls(10 + i)
            torch.cuda.synchronize()
            for _ in range(20):
                for f, _, _ in mine:
                    f(stream)
            (stream or torch.cuda.current_stream()).synchronize()
            for _, out, want in mine:
                assert torch.equal(out, want)
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    for streams in ([None, None, None], [side, side, torch.cuda.Stream()]):
        ts = [threading.Thread(target=work, args=(i, s)) for i, s in enumerate(streams)]
        for t in ts:
            t.start()
        for t in ts:
            t.join()
        assert not errors, errors
    assert dlf_b200.device_status() == 0


def test_operators_in_graphs_that_are_replayed_in_turn():
    """Two graphs and eager calls between them: each call has scratch of its own, and follows its inputs from replay to replay."""
    sets = [_calls(1), _calls(2)]
    graphs = []
    for calls in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            for f, _, _ in calls:
                f(None)
        graphs.append(g)
    for _ in range(3):
        for calls in sets:
            for _, out, _ in calls:
                out.zero_()
        graphs[0].replay()
        sets[1][0][0](None)
        graphs[1].replay()
        graphs[0].replay()
        torch.cuda.synchronize()
        for calls in sets:
            for _, out, want in calls:
                assert torch.equal(out, want)
    assert dlf_b200.device_status() == 0


def test_generation_in_a_graph_follows_lengths_and_positions():
    g = torch.Generator(device="cuda").manual_seed(3)
    table, kp, vp = _cache(g, 2, 64, 16, 2, 64, torch.float16)
    q, k = torch.randn(2, 4, 64, generator=g, device="cuda").half(), torch.randn(2, 2, 64, generator=g, device="cuda").half()
    y, pos, n = torch.empty_like(q), torch.tensor([0, 5], dtype=torch.int32, device="cuda"), torch.tensor([1, 6], dtype=torch.int32, device="cuda")
    gdnn.paged_append(k, k, kp, vp, table, pos)
    gdnn.paged_attention(q, kp, vp, table, n, y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gdnn.paged_append(k, k, kp, vp, table, pos)
        gdnn.paged_attention(q, kp, vp, table, n, y)
        pos.add_(1)
        n.add_(1)
    for step in range(40):
        k.copy_(torch.randn(2, 2, 64, generator=g, device="cuda"))
        at, length = pos.clone(), n.clone()
        graph.replay()
        for i in range(2):
            idx = torch.arange(int(length[i]), device="cuda")
            flat = table[i].long()[idx // 16] * 16 + idx % 16
            kk, vv = kp.reshape(-1, 2, 64)[flat], vp.reshape(-1, 2, 64)[flat]
            assert torch.equal(kk[int(at[i])], k[i])
            want, a, e = _attention_want(q[i:i + 1], kk, vv, torch.ones(len(idx), dtype=torch.bool, device="cuda"), 1 / 8)
            _check_rows(y[i:i + 1], want, a, e, torch.float16, _half_step(torch.float16) ** 2)


def test_callers_scratch_is_used_and_too_little_is_refused():
    calls = _calls(4)
    own = torch.empty(64 << 20, dtype=torch.uint8, device="cuda")
    with gblas.scratch(own):
        for f, out, want in calls:
            out.zero_()
            own.fill_(255)  # (whatever is left there)
            f(None)
            assert torch.equal(out, want)
    with gblas.scratch(torch.empty(16, dtype=torch.uint8, device="cuda")):
        for f, _, _ in calls:
            with pytest.raises(BLASError) as e:
                f(None)
            assert e.value.status == StatusCode.kInsufficientMemoryTemp
    assert dlf_b200.device_status() == 0


@pytest.mark.parametrize("start", [0, 1, 4, 8, 255])
def test_callers_scratch_may_start_anywhere(start):
    """With just what is needed, and nothing written beside it."""
    calls = _calls(6)
    L = dlf_b200.lib()
    needs = [None, L.dlf_b200_attention_workspace_bytes(2, 1, 4000, 8, 2, 64), L.dlf_b200_attention_workspace_bytes(1, 200, 3000, 2, 1, 128),
             L.dlf_b200_paged_attention_workspace_bytes(3, 4, 2, 64)]
    needs[0] = needs[1]  # (the product asks for less)
    for (f, out, want), need in zip(calls, needs):
        own = torch.full((need + 512,), 77, dtype=torch.uint8, device="cuda")
        at = (start - own.data_ptr()) % 256
        out.zero_()
        with gblas.scratch(own[at:at + need]):
            f(None)
        assert torch.equal(out, want)
        assert bool((own[:at] == 77).all()) and bool((own[at + need:] == 77).all())
    assert dlf_b200.device_status() == 0


def test_results_do_not_depend_on_timing():
    calls = _calls(5)
    for _ in range(20):
        for f, out, want in calls:
            f(None)
            assert torch.equal(out, want)


# ---------------------------------------------------------------------------------------------
# together


def test_a_decoder_layers_step():
    """A layer of an encoder-decoder model for one new token of every sequence, each step against its definition on what it was given:
    8-bit products for the projections, the cache, attention over it, attention over the encoder's states."""
    g = torch.Generator(device="cuda").manual_seed(0)
    dtype, b, width, h, hk, d, page = torch.bfloat16, 5, 256, 4, 2, 64, 16
    names = {"q": h * d, "k": hk * d, "v": hk * d, "o": width, "cq": h * d, "co": width}
    weights = {}
    for name, n in names.items():
        k = h * d if name in ("o", "co") else width
        w = torch.randn(n, k, generator=g, device="cuda") / math.sqrt(k)
        weights[name] = tensor.quantize(w)
    states = torch.randn(b, 90, 2, hk, d, generator=g, device="cuda").to(dtype)
    state_lengths = torch.tensor([90, 1, 40, 0, 77], dtype=torch.int32, device="cuda")
    table, kp, vp = _cache(g, b, 100, page, hk, d, dtype)
    n = torch.tensor([1, 100, 33, 16, 17], dtype=torch.int32, device="cuda")

    def project(x, name):
        w, sw = weights[name]
        q, s = tensor.quantize(x)
        want_q, want_s = _quantized(x.cpu())
        assert torch.equal(q.cpu(), want_q) and torch.equal(s.cpu(), want_s)
        y = tensor.matmul_int8(q, s, w, sw, dtype=dtype)
        scaled = (q.double() @ w.double().t()) * sw.double() * s.double().unsqueeze(1)
        assert bool(((y.double() - scaled).abs() <= (_half_step(dtype) + 2.0 ** -22) * scaled.abs()).all())
        return y

    x = torch.randn(b, width, generator=g, device="cuda").to(dtype)
    q, k, v = project(x, "q").view(b, h, d), project(x, "k").view(b, hk, d), project(x, "v").view(b, hk, d)
    gdnn.paged_append(k, v, kp, vp, table, n - 1)
    y = torch.empty_like(q)
    gdnn.paged_attention(q, kp, vp, table, n, y)
    for i in range(b):
        idx = torch.arange(int(n[i]), device="cuda")
        flat = table[i].long()[idx // page] * page + idx % page
        kk, vv = kp.view(-1, hk, d)[flat], vp.view(-1, hk, d)[flat]
        assert torch.equal(kk[-1], k[i]) and torch.equal(vv[-1], v[i])
        want, a, e = _attention_want(q[i:i + 1], kk, vv, torch.ones(len(idx), dtype=torch.bool, device="cuda"), 1 / 8)
        _check_rows(y[i:i + 1], want, a, e, dtype, _half_step(dtype) ** 2)
    x = project(y.view(b, h * d), "o")
    q = project(x, "cq").view(b, 1, h, d)
    y = torch.empty_like(q)
    gdnn.attention(q, states[:, :, 0], states[:, :, 1], y, key_lengths=state_lengths)
    for i in range(b):
        keep = torch.arange(90, device="cuda") < state_lengths[i]
        want, a, e = _attention_want(q[i], states[i, :, 0], states[i, :, 1], keep, 1 / 8)
        _check_rows(y[i], want, a, e, dtype, _half_step(dtype) ** 2)
    project(y.view(b, h * d), "co")
    assert dlf_b200.device_status() == 0


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("cuda_graph", [False, True])
def test_predictor_attention_node(dtype, cuda_graph):
    for three in (False, True):
        g = predict.Graph()
        node = g.append("Attention", q_num_heads=4, kv_num_heads=2)
        dims = [(2, 30, 256), (2, 50, 128), (2, 50, 128)] if three else [(2, 4, 30, 64), (2, 2, 50, 64), (2, 2, 50, 64)]
        for name, d in zip("qkv", dims):
            node.addInput(g.addInput(name, predict.DataType.FLOAT, d))
        for _ in range(3):
            node.addInput(None)
        node.addInput(g.addInput("n", predict.DataType.INT64, (2,)))
        g.addOutput(node.addOutput("y"))
        p = predict.Predictor(g, dtype, cuda_graph=cuda_graph)
        for step in range(4):
            data = [_rand(step * 3 + i, *d).to(dtype) for i, d in enumerate(dims)]
            n = torch.tensor([50 - step, 7 * step])
            for i, x in enumerate(data + [n]):
                p.set(i, x)
            p.predict()
            q, k, v = ((x.view(2, -1, m, 64) if three else x.transpose(1, 2)).cuda() for x, m in zip(data, (4, 2, 2)))
            y = torch.from_numpy(p.get(0)).to(dtype).cuda()
            y = y.view(2, 30, 4, 64) if three else y.transpose(1, 2)
            for i in range(2):
                want, a, e = _attention_want(q[i], k[i], v[i], torch.arange(50, device="cuda") < n[i], 1 / 8)
                _check_rows(y[i], want, a, e, dtype, _half_step(dtype))
    g = predict.Graph()
    node = g.append("Attention")
    for name in "qkv":
        node.addInput(g.addInput(name, predict.DataType.FLOAT, (1, 2, 8, 64)))
    g.addOutput(node.addOutput("y"))
    with pytest.raises(NotImplementedError):
        predict.Predictor(g, torch.float32)


@pytest.mark.parametrize("dtype", TYPES)
def test_predictor_products_in_8_bit_integers(dtype):
    """Gemm (+ bias, + Relu), Gemm with stored transposed weights, MatMul of a batch, against the same layers on what they were given."""
    rng = np.random.default_rng(0)
    w1, b1, w2, w3 = (rng.standard_normal(s).astype(np.float32) for s in ((100, 72), (72,), (40, 72), (40, 24)))

    def build(int8):
        g = predict.Graph()
        n = g.append("Gemm")
        for v in (g.addInput("x", predict.DataType.FLOAT, (30, 100)), g.addInitializer("w1", w1), g.addInitializer("b1", b1)):
            n.addInput(v)
        h1 = n.addOutput("h1")
        if int8:
            n = g.append("Relu")
            n.addInput(h1)
            h1 = n.addOutput("r1")
        n = g.append("Gemm", transB=1)
        n.addInput(h1)
        n.addInput(g.addInitializer("w2", w2))
        h2 = n.addOutput("h2")
        n = g.append("MatMul")
        n.addInput(h2)
        n.addInput(g.addInitializer("w3", w3))
        for v in (h1, h2, n.addOutput("y")):
            g.addOutput(v)
        return predict.Predictor(g, dtype, int8=int8)

    p = build(True)
    assert [type(op).__name__ for op in p.operators] == ["Int8ProductOp"] * 3
    x = _rand(1, 30, 100).to(dtype)
    for _ in range(3):  # launch by launch, captured, replayed
        p.set(0, x)
        p.predict()
        h1, h2, y = (torch.from_numpy(p.get(i)).to(dtype) for i in range(3))
        for given, w, bias, relu, got in ((x, torch.from_numpy(w1).t(), torch.from_numpy(b1), True, h1), (h1, torch.from_numpy(w2), None, False, h2),
                                          (h2, torch.from_numpy(w3).t(), None, False, y)):
            qa, sa = _quantized(given)
            qw, sw = _quantized(w.to(dtype).contiguous())
            scaled = (qa.double() @ qw.double().t()) * sa.double().unsqueeze(1) * sw.double()
            want = scaled + (bias.to(dtype).double() if bias is not None else 0)
            want = want.clamp_min(0) if relu else want
            tol = 3 * 2.0 ** -24 * (scaled.abs() + want.abs()) + _half_step(dtype) * want.abs() * (1 + 2.0 ** -20)
            assert bool(((got.double() - want).abs() <= tol).all())
    assert [type(op).__name__ for op in build(False).operators] == ["GemmOp", "GemmOp", "MatMulOp"]


@pytest.mark.parametrize("dtype", HALF)
def test_predictor_8_bit_product_behind_channels_last_convolutions(dtype):
    """Convolutions whose values stay channels-last, Flatten, Gemm: what the product is given is in the graph's order."""
    rng = np.random.default_rng(1)
    wc, wg = rng.standard_normal((16, 8, 3, 3)).astype(np.float32), rng.standard_normal((16 * 36, 24)).astype(np.float32)

    def build(int8):
        g = predict.Graph()
        n = g.append("Conv", kernel_shape=(3, 3), pads=(1, 1, 1, 1))
        n.addInput(g.addInput("x", predict.DataType.FLOAT, (2, 8, 6, 6)))
        n.addInput(g.addInitializer("wc", wc))
        h = n.addOutput("h")
        n = g.append("Flatten")
        n.addInput(h)
        f = n.addOutput("f")
        n = g.append("Gemm")
        n.addInput(f)
        n.addInput(g.addInitializer("wg", wg))
        for v in (f, n.addOutput("y")):
            g.addOutput(v)
        return predict.Predictor(g, dtype, int8=int8)

    x = _rand(3, 2, 8, 6, 6).to(dtype)
    p, plain = build(True), build(False)
    for _ in range(3):
        for r in (p, plain):
            r.set(0, x)
            r.predict()
        given, got = (torch.from_numpy(p.get(i)).to(dtype) for i in range(2))
        assert torch.equal(given, torch.from_numpy(plain.get(0)).to(dtype))
        qa, sa = _quantized(given)
        qw, sw = _quantized(torch.from_numpy(wg).t().to(dtype).contiguous())
        want = (qa.double() @ qw.double().t()) * sa.double().unsqueeze(1) * sw.double()
        tol = 3 * 2.0 ** -24 * 2 * want.abs() + _half_step(dtype) * want.abs() * (1 + 2.0 ** -20)
        assert bool(((got.double() - want).abs() <= tol).all())


# ---------------------------------------------------------------------------------------------
# far addresses


def test_rows_and_pages_beyond_32_bit_offsets():
    """A cache and rows whose last elements lie more than 2^32 bytes (and 2^31 elements) behind the first."""
    free, _ = torch.cuda.mem_get_info()
    if free < 40 << 30:
        pytest.skip("not enough free memory")
    page, hk, d = 16, 8, 128
    pages = (1 << 31) // (page * hk * d) + 2000
    kp = torch.empty(pages, page, hk, d, dtype=torch.float16, device="cuda")
    vp = torch.empty_like(kp)
    table = torch.arange(pages - 20, pages, dtype=torch.int32, device="cuda").view(1, 20)
    kp[-20:], vp[-20:] = torch.randn(20, page, hk, d, device="cuda"), torch.randn(20, page, hk, d, device="cuda")
    new = torch.randn(1, hk, d, device="cuda").half()
    gdnn.paged_append(new, new, kp, vp, table, torch.tensor([319], dtype=torch.int32, device="cuda"))
    assert torch.equal(kp[-1, -1], new[0]) and torch.equal(vp[-1, -1], new[0])
    q = torch.randn(1, 16, d, device="cuda").half()
    y = torch.empty_like(q)
    gdnn.paged_attention(q, kp, vp, table, torch.tensor([320], dtype=torch.int32, device="cuda"), y)
    k, v = kp[-20:].view(1, -1, hk, d), vp[-20:].view(1, -1, hk, d)
    want, a, e = _attention_want(q, k[0], v[0], torch.ones(320, dtype=torch.bool, device="cuda"), 1 / math.sqrt(d))
    _check_rows(y, want, a, e, torch.float16, _half_step(torch.float16) ** 2)
    # two entries of a batch, that far apart
    far = kp.view(-1)[: pages * page * hk * d].as_strided((2, 200, hk, d), ((1 << 31) + (1 << 20), hk * d, d, 1))
    far[0], far[1] = torch.randn(200, hk, d, device="cuda"), torch.randn(200, hk, d, device="cuda")
    for lq in (1, 100):
        q = torch.randn(2, lq, hk, d, device="cuda").half()
        y = torch.empty_like(q)
        gdnn.attention(q, far, far, y)
        for i in range(2):
            want, a, e = _attention_want(q[i], far[i], far[i], torch.ones(200, dtype=torch.bool, device="cuda"), 1 / math.sqrt(d))
            _check_rows(y[i], want, a, e, torch.float16, _half_step(torch.float16) if lq > 32 else _half_step(torch.float16) ** 2)
    del kp, vp, far, k, v
    rows = torch.zeros(3, (1 << 31) + 64, dtype=torch.int8, device="cuda")  # products whose lines lie that far apart
    a = rows[:, :200]
    a.copy_(torch.randint(-99, 99, (3, 200), dtype=torch.int8))
    s = torch.ones(3, device="cuda")
    assert torch.equal(tensor.matmul_int8(a, s, a, s).double(), a.double() @ a.double().t())
    rows[:, :32].zero_()
    x = rows.view(torch.float16)[:, :100]
    x.copy_(_rand(1, 3, 100))
    q8, sc = tensor.quantize(x)
    want_q, want_s = _quantized(x.cpu())
    assert torch.equal(q8.cpu(), want_q) and torch.equal(sc.cpu(), want_s)
