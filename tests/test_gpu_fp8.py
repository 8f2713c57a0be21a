"""The block-scaled 8-bit products (fp8_quantize, fp8_gemm, fp8_linear) against their formulas in 64 bits."""
import ctypes as C
import importlib

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
pkg = importlib.import_module("ferrum-torrens_b200")
L = pkg._lib

E4M3 = torch.float8_e4m3fn
DT = {"bf16": torch.bfloat16, "f32": torch.float32}
DEV = "cuda:0"


@pytest.fixture(scope="module")
def moe():
    m = pkg.B200MoE(0, pkg.ExpertShapes(64, 16), 1, experts=1, layers=1, top_k=1, shared_inter=16, max_tokens=1)
    yield m
    m.close()


def rng(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def activations(seed, m, k, dtype, pad=0, offset=0):
    """[m, k] whose rows are k + pad apart and start `offset` elements into their buffer."""
    buf = torch.randn((m, k + pad), generator=rng(seed), device=DEV) * torch.exp2(3 * torch.randn((m, 1), generator=rng(seed + 1), device=DEV))
    return buf.to(dtype)[:, offset:offset + k]


def weight(seed, n, k):
    w = (torch.randn((n, k), generator=rng(seed), device=DEV) * 90).clamp(-448, 448).to(E4M3)
    s = torch.exp2(torch.randn((-(-n // 128), -(-k // 128)), generator=rng(seed + 7), device=DEV)) * 1e-3
    return w, s


# ------------------------------------------------------------------ the formulas, in 64 bits on the CPU
def e4m3_nearest(y):
    """The e4m3 value nearest to each y, ties to even, saturating."""
    step = np.exp2(np.floor(np.log2(np.maximum(np.abs(y), 2.0 ** -6))) - 3)
    return np.clip(np.round(y / step) * step, -448, 448)


def quantised(x):
    """(codes' values [M, K], scales [blocks, M]): the three roundings to f32 are the definition's."""
    x = x.double().cpu().numpy()
    m, k = x.shape
    q, scales = np.zeros((m, k)), []
    with np.errstate(invalid="ignore", over="ignore"):
        for b in range(0, k, 128):
            v = x[:, b:b + 128]
            a0 = np.maximum(np.nan_to_num(np.abs(v), nan=0.0, posinf=np.inf).max(1), 448 * 2.0 ** -126).astype(np.float32).astype(np.float64)
            inv = (448.0 / a0).astype(np.float32).astype(np.float64)
            y = (v * inv[:, None]).astype(np.float32).astype(np.float64)
            q[:, b:b + 128] = np.where(np.isnan(y), np.nan, e4m3_nearest(np.nan_to_num(y)))
            scales.append((a0 / 448.0).astype(np.float32))
    return q, np.stack(scales)


def product(q, scales, w, ws):
    """(c, S) in 64 bits: S the sum of the terms' magnitudes, which the rounding errors go by."""
    w, ws = w.float().double().cpu().numpy(), ws.double().cpu().numpy()
    c, mag = 0.0, 0.0
    for b in range(scales.shape[0]):
        at = slice(128 * b, 128 * b + 128)
        rows = q[:, at] * scales[b].astype(np.float64)[:, None]
        cols = w[:, at] * np.repeat(ws[:, b], 128)[:w.shape[0], None]
        c, mag = c + rows @ cols.T, mag + np.abs(rows) @ np.abs(cols).T
    return c, mag


def check_product(got, q, scales, w, ws):
    c, mag = product(q, scales, w, ws)
    blocks = scales.shape[0]
    # products of e4m3 are exact in f32; 128 additions of a block, one per block, the product of the two scales and its
    # multiplication: each off by at most one step 2^-23 (a tensor core may cut off where an ALU rounds)
    tol = (128 + blocks + 3) * 2.0 ** -23 * mag + np.abs(c) * torch.finfo(got.dtype).eps / 2 + 1e-38
    d = np.abs(got.double().cpu().numpy() - c)
    assert (d <= tol).all(), (float((d / tol).max()), np.unravel_index(np.argmax(d / tol), d.shape))


# ------------------------------------------------------------------ quantisation
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("m,k,pad,offset", [(1, 16, 0, 0), (1, 128, 0, 0), (2, 144, 0, 0), (7, 1040, 16, 8), (37, 2048, 0, 0), (9, 2000, 5, 3),
                                            (8, 256, 1, 1), (300, 4096, 0, 0), (1, 16, 1, 1)])
def test_quantize_is_the_formula_bit_for_bit(moe, m, k, pad, offset, dtype):
    x = activations(m * 1000 + k, m, k, DT[dtype], pad, offset)
    q, s = moe.fp8_quantize(x)
    want_q, want_s = quantised(x)
    assert np.array_equal(s.cpu().numpy(), want_s)
    assert np.array_equal(q.float().cpu().numpy(), want_q.astype(np.float32))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("m,k,pad", [(5000, 2064, 0), (1203, 8192, 8), (4999, 144, 3)])
def test_quantize_walks_over_large_inputs(moe, m, k, pad, dtype):
    x = activations(m + k, m, k, DT[dtype], pad)
    q, s = moe.fp8_quantize(x)
    want_q, want_s = quantised(x)
    assert np.array_equal(s.cpu().numpy(), want_s)
    assert np.array_equal(q.float().cpu().numpy(), want_q.astype(np.float32))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_quantize_special_values(moe, dtype):
    big, tiny = torch.finfo(DT[dtype]).max, torch.finfo(DT[dtype]).smallest_normal
    rows = torch.zeros((8, 272))
    rows[0] = 0.0
    rows[1] = tiny / 4                                   # all subnormal
    rows[2, ::3], rows[2, 5] = big, -big
    rows[3] = torch.arange(272) - 135.5
    rows[4] = 1.0
    rows[4, 7], rows[4, 130] = float("nan"), float("nan")     # a NaN is one element's matter
    rows[5] = 2.0
    rows[5, 3] = float("inf")                            # an infinity is its block's
    rows[5, 4] = float("-inf")
    rows[6, :128] = 448.0
    rows[6, :16] = torch.tensor([17., 18., 19., 20., 21., 22., 23., 1.0625, 1.1875, 2.0 ** -10, 3 * 2.0 ** -10, 2.0 ** -9, 447., 432., 440., -0.0])
    rows[7, 128:] = -tiny
    x = rows.to(DT[dtype]).to(DEV)
    q, s = moe.fp8_quantize(x)
    want_q, want_s = quantised(x)
    assert np.array_equal(s.cpu().numpy(), want_s)
    assert np.array_equal(q.float().cpu().numpy(), want_q.astype(np.float32), equal_nan=True)
    assert np.isinf(want_s[0, 5]) and np.isnan(want_q[5, 3:5]).all() and (want_q[5, 5:128] == 0).all()
    assert want_s[0, 0] == 2.0 ** -126


def test_quantize_writes_its_rows_only_and_reaches_past_32_bits(moe):
    m, k = 2 ** 20 + 3, 2048
    x = torch.empty((m, k), dtype=torch.bfloat16, device=DEV)
    x[-3:] = activations(5, 3, k, torch.bfloat16)
    x[:3] = x[-3:]
    q = torch.empty((m + 2, k), dtype=torch.uint8, device=DEV)
    q[-2:] = 0xa5
    s = torch.full((16 * m + 5,), -7.0, device=DEV)
    moe.fp8_quantize(x, out=(q[:m].view(E4M3), s[:16 * m].view(16, m)))
    want_q, want_s = quantised(x[-3:])
    assert np.array_equal(q[m - 3:m].view(E4M3).float().cpu().numpy(), want_q.astype(np.float32))
    assert np.array_equal(s[:16 * m].view(16, m)[:, -3:].cpu().numpy(), want_s)
    assert (q[-2:] == 0xa5).all() and (s[16 * m:] == -7.0).all()


# ------------------------------------------------------------------ products
SHAPES = [(1, 1, 16), (1, 128, 128), (2, 129, 144), (3, 5, 4112), (8, 2048, 512), (15, 640, 2048), (16, 64, 2048), (16, 300, 8192), (17, 130, 272),
          (31, 1000, 128), (33, 300, 1040), (64, 512, 512), (65, 257, 2048), (100, 2048, 4096), (127, 127, 112), (128, 128, 128), (129, 384, 640),
          (200, 1000, 2000), (256, 256, 256), (300, 4100, 400), (513, 768, 1152), (1000, 2050, 2064), (2100, 520, 384)]


@pytest.mark.parametrize("out", ["bf16", "f32"])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_gemm(moe, m, n, k, out):
    q, s = moe.fp8_quantize(activations(m + n, m, k, torch.float32))
    w, ws = weight(k + n, n, k)
    buf = torch.full((m + 1, n + 3), 77.0, dtype=DT[out], device=DEV)
    c = buf[:m, :n]                                      # rows apart; what is behind a row and behind the last row stays
    moe.fp8_gemm(q, s, w, ws, c)
    check_product(c, q.double().cpu().numpy(), s.cpu().numpy(), w, ws)
    assert (buf[:, n:] == 77.0).all() and (buf[m] == 77.0).all()
    again = torch.empty((m, n), dtype=DT[out], device=DEV)
    moe.fp8_gemm(q, s, w, ws, again)
    assert torch.equal(again, c), "the same inputs give the same bits"
    moe.sync_status()


@pytest.mark.parametrize("x,out", [("bf16", "bf16"), ("bf16", "f32"), ("f32", "bf16"), ("f32", "f32")])
@pytest.mark.parametrize("m,n,k,pad,offset", [(1, 2048, 2048, 0, 0), (1, 1, 16, 0, 0), (4, 300, 2000, 8, 0), (7, 1025, 4096, 3, 1), (13, 256, 144, 0, 0),
                                              (16, 5000, 512, 0, 0), (16, 136, 8192, 0, 0), (5, 200, 8208, 0, 0), (17, 520, 1024, 0, 0), (64, 384, 2048, 8, 8),
                                              (140, 260, 640, 1, 0)])
def test_linear_is_the_product_of_the_quantised_rows(moe, m, n, k, pad, offset, x, out):
    rows = activations(m + 3 * k, m, k, DT[x], pad, offset)
    w, ws = weight(n, n, k)
    buf = torch.full((m + 1, n + 5), 77.0, dtype=DT[out], device=DEV)
    c = moe.fp8_linear(rows, w, ws, buf[:m, :n])
    q, s = quantised(rows)
    check_product(c, q, s, w, ws)
    assert (buf[:, n:] == 77.0).all() and (buf[m] == 77.0).all()
    again = torch.empty((m, n), dtype=DT[out], device=DEV)
    scratch = (torch.empty((m, k), dtype=E4M3, device=DEV), torch.empty((-(-k // 128), m), device=DEV))
    moe.fp8_linear(rows, w, ws, again, scratch=scratch)
    assert torch.equal(again, c)
    moe.sync_status()


@pytest.mark.parametrize("m,n,k", [(1, 40000, 2048), (2, 20000, 8192), (4, 10240, 8192), (5, 2048, 8192), (8, 2048, 4096), (12, 100, 2048), (13, 2048, 4096), (16, 8192, 512),
                                   (16, 1000, 8192), (16, 60000, 1040)])
def test_one_kernel_and_two_give_the_same_bits(moe, m, n, k):
    x = activations(m + n, m, k, torch.bfloat16).contiguous()
    w, ws = weight(n + k, n, k)
    c = torch.full((3, m, n), 77.0, device=DEV)
    scratch = moe.fp8_quantize(torch.zeros_like(x))
    lib, p, st = L.lib(), lambda t: C.c_void_p(t.data_ptr()), C.c_void_p(torch.cuda.current_stream().cuda_stream)
    call = lambda q, s, out: lib.ftm_fp8_linear(moe._h, p(x), L.BF16, k, p(w), p(ws), m, n, k, q, s, p(out), L.F32, n, st)
    assert call(C.c_void_p(0), C.c_void_p(0), c[0]) == L.OK
    assert call(p(scratch[0]), p(scratch[1]), c[1]) == L.OK
    moe.fp8_gemm(*moe.fp8_quantize(x), w, ws, c[2])
    assert torch.equal(c[0], c[1]) and torch.equal(c[0], c[2])
    check_product(c[0], *quantised(x), w, ws)
    moe.sync_status()


@pytest.mark.parametrize("sms", [1, 2, 7, 40])
@pytest.mark.parametrize("m", [3, 30, 50, 120, 300, 700])
def test_few_sms(moe, m, sms):
    """A budget of SMs: few CTAs walk over many tiles, and the blocks are split less or not at all."""
    n, k = 1500, 1040
    x = activations(m, m, k, torch.bfloat16).contiguous()
    w, ws = weight(m + 1, n, k)
    q, s = quantised(x)
    moe.set_sm_budget(sms)
    try:
        for out in (torch.float32, torch.bfloat16):
            c = torch.full((m, n), 77.0, dtype=out, device=DEV)
            moe.fp8_linear(x, w, ws, c)
            check_product(c, q, s, w, ws)
            c2 = torch.empty_like(c)
            moe.fp8_gemm(*moe.fp8_quantize(x), w, ws, c2)
            check_product(c2, q, s, w, ws)
        moe.sync_status()
    finally:
        moe.set_sm_budget(0)


@pytest.mark.parametrize("out", ["bf16", "f32"])
@pytest.mark.parametrize("n,ld,offset", [(512, 512, 0), (512, 520, 0), (512, 516, 0), (515, 517, 1), (514, 522, 2), (300, 301, 0), (600, 604, 4)])
def test_output_rows_of_any_alignment(moe, n, ld, offset, out):
    m, k = 400, 256
    q, s = moe.fp8_quantize(activations(n, m, k, torch.bfloat16))
    w, ws = weight(ld, n, k)
    buf = torch.full((m * ld + offset + 9,), 77.0, dtype=DT[out], device=DEV)
    c = buf[offset:].as_strided((m, n), (ld, 1), storage_offset=offset)
    moe.fp8_gemm(q, s, w, ws, c)
    check_product(c, q.double().cpu().numpy(), s.cpu().numpy(), w, ws)
    kept = torch.ones_like(buf, dtype=torch.bool)
    kept.as_strided((m, n), (ld, 1), storage_offset=offset).fill_(False)
    assert (buf[kept] == 77.0).all()


@pytest.fixture(params=[0, 20])
def sms(request, moe):
    """All SMs, or so few that many rows are taken by pairs of them in tiles of 256 x 256."""
    moe.set_sm_budget(request.param)
    yield request.param
    moe.set_sm_budget(0)


@pytest.mark.parametrize("out", ["bf16", "f32"])
@pytest.mark.parametrize("n,ld,offset", [(1281, 1281, 0), (1407, 1407, 1), (1409, 1411, 0), (1534, 1534, 0), (1535, 1537, 3), (1539, 1540, 2), (1343, 1346, 0), (1280, 1284, 4)])
def test_rows_that_start_and_end_anywhere(moe, sms, n, ld, offset, out):
    """Outputs of odd sizes, with ends of every length."""
    m, k = 1100, 128
    q, s = moe.fp8_quantize(activations(n, m, k, torch.bfloat16))
    w, ws = weight(ld, n, k)
    buf = torch.full((m * ld + offset + 9,), 77.0, dtype=DT[out], device=DEV)
    c = buf.as_strided((m, n), (ld, 1), storage_offset=offset)
    moe.fp8_gemm(q, s, w, ws, c)
    check_product(c, q.double().cpu().numpy(), s.cpu().numpy(), w, ws)
    kept = torch.ones_like(buf, dtype=torch.bool)
    kept.as_strided((m, n), (ld, 1), storage_offset=offset).fill_(False)
    assert (buf[kept] == 77.0).all()
    moe.sync_status()


@pytest.mark.parametrize("m,n,k", [(1000, 4100, 2000), (1025, 4097, 272), (600, 9000, 1040), (4097, 1025, 640), (257, 20000, 144)])
def test_pairs_of_sms(moe, sms, m, n, k):
    q, s = moe.fp8_quantize(activations(m + n, m, k, torch.float32))
    w, ws = weight(k + n, n, k)
    for out in (torch.bfloat16, torch.float32):
        c = torch.full((m + 1, n), 77.0, dtype=out, device=DEV)
        moe.fp8_gemm(q, s, w, ws, c[:m])
        check_product(c[:m], q.double().cpu().numpy(), s.cpu().numpy(), w, ws)
        assert (c[m] == 77.0).all()
    moe.sync_status()


@pytest.mark.parametrize("m", [300, 1100])
def test_special_codes_in_tiles_of_pairs(moe, sms, m):
    """A NaN code is its weight row's matter, an infinite scale its token's."""
    n, k = 1400, 400
    q, s = moe.fp8_quantize(activations(3, m, k, torch.bfloat16))
    w, ws = weight(4, n, k)
    clean = torch.empty((m, n), device=DEV)
    moe.fp8_gemm(q, s, w, ws, clean)
    wb, s2 = w.clone().view(torch.uint8), s.clone()
    wb[1333, 399], s2[1, m // 2] = 0x7f, float("inf")
    got = torch.empty_like(clean)
    moe.fp8_gemm(q, s2, wb.view(E4M3), ws, got)
    got, clean = got.cpu().numpy(), clean.cpu().numpy()
    assert np.isnan(got[:, 1333]).all() and not np.isfinite(got[m // 2]).any()
    rows, cols = np.arange(m) != m // 2, np.arange(n) != 1333
    assert np.array_equal(got[np.ix_(rows, cols)], clean[np.ix_(rows, cols)])
    moe.sync_status()


@pytest.mark.parametrize("m", [1, 9, 40, 130, 600])
def test_special_codes_stay_in_their_row_or_column(moe, m):
    n, k = 300, 400
    x = activations(3, m, k, torch.bfloat16)
    w, ws = weight(4, n, k)
    clean = torch.empty((m, n), dtype=torch.float32, device=DEV)
    moe.fp8_linear(x, w, ws, clean)
    wb = w.clone().view(torch.uint8)
    wb[77, 399] = 0x7f                                   # NaN code in the last, short block
    wb[78] = 0x80                                        # a row of -0
    ws2 = ws.clone()
    ws2[2, 1] = 0.0
    x2 = x.clone()
    x2[m // 2, 130] = float("inf")
    got = torch.empty_like(clean)
    moe.fp8_linear(x2, wb.view(E4M3), ws2, got)
    got, clean = got.cpu().numpy(), clean.cpu().numpy()
    assert np.isnan(got[:, 77]).all() and np.isnan(got[m // 2]).all()
    keep = [r for r in range(m) if r != m // 2]
    assert (got[keep, 78] == 0).all()
    cols = [j for j in range(256) if j not in (77, 78)]
    assert np.array_equal(got[np.ix_(keep, cols)], clean[np.ix_(keep, cols)])
    assert np.isfinite(got[keep][:, 256:]).all()


@pytest.mark.parametrize("m", [4, 40, 200])
def test_largest_codes_and_scales(moe, m):
    """Sums of 448 * 448 terms, and scales whose product leaves f32's range only where the result does."""
    n, k = 140, 2048
    x = torch.full((m, k), 3.0e38, device=DEV)
    x[:, ::2] *= -1.0
    x[:, 0] = 3.0e38
    w = torch.full((n, k), 448.0, device=DEV).to(E4M3)
    ws = torch.full((2, 16), 1e-30, device=DEV)
    c = torch.empty((m, n), device=DEV)
    moe.fp8_linear(x, w, ws, c)
    q, s = quantised(x)
    check_product(c, q, s, w, ws)


def test_gemm_output_rows_past_32_bits(moe):
    m, n, k, ld = 9, 64, 128, 2 ** 28 + 1
    q, s = moe.fp8_quantize(activations(1, m, k, torch.bfloat16))
    w, ws = weight(2, n, k)
    buf = torch.empty((8 * ld + n,), dtype=torch.bfloat16, device=DEV)
    c = buf.as_strided((m, n), (ld, 1))
    moe.fp8_gemm(q, s, w, ws, c)
    check_product(c, q.double().cpu().numpy(), s.cpu().numpy(), w, ws)


def test_graphs_streams_and_chained_calls(moe):
    """Captured and replayed on new inputs, twice at once on two streams, and quantise -> product without a wait between."""
    m, n, k = 12, 1000, 2048
    w, ws = weight(1, n, k)
    w2, ws2 = weight(2, 300, 1008)
    inputs = [activations(i, m, k, torch.bfloat16).contiguous() for i in range(4)]

    def want(x):
        c = torch.empty((m, n), device=DEV)
        moe.fp8_linear(x, w, ws, c)
        return c
    wanted = [want(x) for x in inputs]
    x, c = inputs[0].clone(), torch.empty((m, n), device=DEV)
    y, big = activations(9, 300, 1008, torch.float32), torch.empty((300, 300), dtype=torch.bfloat16, device=DEV)
    scratch = tuple(t.clone() for t in moe.fp8_quantize(y))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        moe.fp8_linear(x, w, ws, c, scratch=tuple(t.clone() for t in moe.fp8_quantize(x)))
        moe.fp8_quantize(y, out=scratch)
        moe.fp8_gemm(*scratch, w2, ws2, big)
    for i in (1, 2, 3):
        x.copy_(inputs[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(c, wanted[i])
    q, s = quantised(y)
    check_product(big, q, s, w2, ws2)
    streams, outs = [torch.cuda.Stream() for _ in range(3)], [torch.empty((m, n), device=DEV) for _ in range(3)]
    torch.cuda.synchronize()
    for _ in range(20):
        for st, x_in, o in zip(streams, inputs, outs):
            with torch.cuda.stream(st):
                moe.fp8_linear(x_in, w, ws, o)
    torch.cuda.synchronize()
    for o, v in zip(outs, wanted):
        assert torch.equal(o, v)
    moe.sync_status()


def test_scratch_made_for_another_stream_is_not_handed_out_early(moe):
    """Without scratch of its own a call on a side stream must not see it reused by what the current stream allocates meanwhile."""
    m, n, k = 64, 256, 2048
    x, (w, ws) = activations(1, m, k, torch.bfloat16), weight(2, n, k)
    want = torch.empty((m, n), device=DEV)
    moe.fp8_linear(x, w, ws, want)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for given in (side, side.cuda_stream):
        c = torch.zeros((m, n), device=DEV)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.cuda._sleep(20_000_000)
        moe.fp8_linear(x, w, ws, c, stream=given)
        q, s = moe.fp8_quantize(x, stream=given)
        del q, s
        junk = [torch.full((m, k), 0x7f, dtype=torch.uint8, device=DEV) for _ in range(8)] + [torch.full((k // 128, m), 9e9, device=DEV) for _ in range(8)]
        torch.cuda.synchronize()
        assert torch.equal(c, want) and len(junk) == 16
    # an adapter with a stream of its own takes the default stream's place
    own = pkg.B200MoE(0, pkg.ExpertShapes(64, 16), 1, experts=1, layers=1, top_k=1, shared_inter=16, max_tokens=1, stream=side)
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
    c = torch.zeros((m, n), device=DEV)
    side.wait_stream(torch.cuda.current_stream())
    own.fp8_linear(x, w, ws, c)
    junk = [torch.full((m, k), 0x7f, dtype=torch.uint8, device=DEV) for _ in range(8)]
    torch.cuda.synchronize()
    assert torch.equal(c, want) and junk
    own.close()


def test_refusals(moe):
    x = torch.zeros((4, 256), dtype=torch.bfloat16, device=DEV)
    w, ws = weight(0, 130, 256)
    q, s = moe.fp8_quantize(x)
    c = torch.empty((4, 130), device=DEV)
    bad = [
        lambda: moe.fp8_quantize(x.half()), lambda: moe.fp8_quantize(x[:, :250]), lambda: moe.fp8_quantize(x.cpu()), lambda: moe.fp8_quantize(x[0]),
        lambda: moe.fp8_quantize(x.t()), lambda: moe.fp8_quantize(x[:0]), lambda: moe.fp8_quantize(x[:, :0]), lambda: moe.fp8_quantize(x[:1].expand(4, 256)),
        lambda: moe.fp8_quantize(x, out=(q, s.t().contiguous())), lambda: moe.fp8_quantize(x, out=(q.view(torch.uint8), s)),
        lambda: moe.fp8_gemm(q, s, w, ws[:1].contiguous(), c), lambda: moe.fp8_gemm(q, s, w[:, :240].contiguous(), ws, c),
        lambda: moe.fp8_gemm(q, s[:1].contiguous(), w, ws, c), lambda: moe.fp8_gemm(q, s, w, ws.bfloat16(), c), lambda: moe.fp8_gemm(q, s, w, ws, c.half()),
        lambda: moe.fp8_gemm(q, s, w, ws, c[:3]), lambda: moe.fp8_gemm(q, s, w, ws, c.t()), lambda: moe.fp8_gemm(q, s, w, ws, c[:1].expand(4, 130)),
        lambda: moe.fp8_gemm(x, s, w, ws, c), lambda: moe.fp8_gemm(q, s, w.t(), ws, c), lambda: moe.fp8_linear(x.cpu(), w, ws, c),
        lambda: moe.fp8_linear(x, w, ws, c, scratch=(q[:2].contiguous(), s)), lambda: moe.fp8_linear(x[:, :128], w, ws, c),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(pkg.MoEError) as e:
            call()
        assert e.value.kind == "Bad", i
    lib, h, p = L.lib(), moe._h, lambda t, off=0: C.c_void_p(t.data_ptr() + off)
    null, st = C.c_void_p(0), C.c_void_p(0)
    gemm = lambda a=p(q), sa=p(s), pw=p(w), sw=p(ws), m=4, n=130, k=256, pc=p(c), dt=L.F32, ld=130: lib.ftm_fp8_gemm(h, a, sa, pw, sw, m, n, k, pc, dt, ld, st)
    assert gemm() == L.OK
    for kw in (dict(a=null), dict(sa=null), dict(pw=null), dict(sw=null), dict(pc=null), dict(m=0), dict(m=-1), dict(n=0), dict(k=0), dict(k=248), dict(k=-16),
               dict(dt=L.I32), dict(ld=129), dict(a=p(q, 8)), dict(pw=p(w, 1)), dict(pc=p(c, 2)), dict(sa=p(s, 2)), dict(sw=p(ws, 1))):
        assert gemm(**kw) == L.ERR_BAD, kw
    quant = lambda px=p(x), dt=L.BF16, m=4, k=256, ld=256, pq=p(q), ps=p(s): lib.ftm_fp8_quantize(h, px, dt, m, k, ld, pq, ps, st)
    assert quant() == L.OK
    for kw in (dict(px=null), dict(pq=null), dict(ps=null), dict(dt=L.I64), dict(m=0), dict(k=8), dict(ld=255), dict(px=p(x, 1)), dict(pq=p(q, 4)), dict(ps=p(s, 1))):
        assert quant(**kw) == L.ERR_BAD, kw
    linear = lambda px=p(x), dt=L.BF16, ld=256, pw=p(w), sw=p(ws), m=4, n=130, k=256, pq=null, ps=null, pc=p(c), ct=L.F32, cl=130: lib.ftm_fp8_linear(
        h, px, dt, ld, pw, sw, m, n, k, pq, ps, pc, ct, cl, st)
    assert linear() == L.OK
    many = torch.zeros((17, 256), dtype=torch.bfloat16, device=DEV)
    cm, (qm, sm) = torch.empty((17, 130), device=DEV), moe.fp8_quantize(many)
    big = dict(px=p(many), m=17, pc=p(cm))
    assert linear(**big, pq=p(qm), ps=p(sm)) == L.OK
    for kw in (dict(px=null), dict(pw=null), dict(sw=null), dict(pc=null), dict(m=0), dict(n=0), dict(k=0), dict(k=8), dict(dt=L.I32), dict(ct=L.I64), dict(ld=255),
               dict(cl=129), dict(pw=p(w, 8)), dict(px=p(x, 1)), dict(m=2 ** 30 + 1), dict(n=2 ** 30 + 1, cl=2 ** 31), dict(k=2 ** 30 + 16, ld=2 ** 31),
               big, dict(**big, pq=p(qm)), dict(**big, ps=p(sm)), dict(**big, pq=p(qm, 8), ps=p(sm)), dict(**big, pq=p(qm), ps=p(sm, 2))):
        assert linear(**kw) == L.ERR_BAD, kw
    assert lib.ftm_fp8_gemm(null, null, null, null, null, 1, 1, 16, null, 0, 1, null) == L.ERR_BAD
    torch.cuda.synchronize()


def test_calls_from_several_threads(moe):
    """Kernels of every kind beside one another, from host threads with a stream each, give what they give alone."""
    import threading
    gen = rng(11)
    pk = torch.randint(-2 ** 31, 2 ** 31 - 1, (128, 4096), generator=gen, device=DEV, dtype=torch.int32)
    sk = torch.randint(0x20, 0x40, (64, 4096), generator=gen, device=DEV, dtype=torch.uint8)
    glob = torch.full((4096,), 0x3c00, device=DEV, dtype=torch.int16)
    act = activations(5, 64, 1024, torch.bfloat16).contiguous()
    logits, ids = activations(6, 40, 30001, torch.float32), torch.arange(40, device=DEV)
    jobs = []
    for i, (m, n, k) in enumerate([(1000, 4100, 2000), (100, 4096, 2048), (13, 2048, 4096), (64, 10240, 512), (1500, 2000, 1024), (30, 3000, 2048)]):
        x, (w, ws) = activations(i, m, k, torch.bfloat16).contiguous(), weight(i + 1, n, k)
        scratch = moe.fp8_quantize(x)

        def linear(stream, x=x, w=w, ws=ws, scratch=scratch, c=torch.empty((m, n), device=DEV)):
            return [moe.fp8_linear(x, w, ws, c, scratch=scratch, stream=stream)]
        jobs.append(linear)
    out = moe.logprobs(logits, ids, 9)
    jobs.append(lambda stream: list(moe.logprobs(logits, ids, 9, out=out, stream=stream)))
    c = torch.empty((64, 4096), device=DEV)
    jobs.append(lambda stream: [moe.dense_gemv(act, pk, sk, glob, c, stream=stream)])
    alone = []
    for job in jobs:
        alone.append([t.clone() for t in job(torch.cuda.current_stream())])
    torch.cuda.synchronize()
    failures = []

    def work(job, want):
        stream = torch.cuda.Stream(device=0)
        try:
            for _ in range(5):
                for _ in range(20):
                    got = job(stream)
                stream.synchronize()
                for a, b in zip(got, want):
                    if not torch.equal(a.view(torch.int32), b.view(torch.int32)):
                        failures.append("another result")
        except Exception as e:
            failures.append(repr(e))
    threads = [threading.Thread(target=work, args=a) for a in zip(jobs, alone)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures, failures
    moe.sync_status()


@pytest.mark.parametrize("m,n,k", [(5, 600, 1024), (40, 600, 1024), (1000, 4100, 2000)])
def test_first_call_of_a_host_thread(moe, m, n, k):
    """A thread in which nothing has used CUDA yet."""
    import threading
    x, (w, ws) = activations(1, m, k, torch.bfloat16).contiguous(), weight(2, n, k)
    q, s = moe.fp8_quantize(x)
    want, c = torch.empty((m, n), device=DEV), torch.zeros((2, m, n), device=DEV)
    moe.fp8_gemm(q, s, w, ws, want)
    stream = torch.cuda.current_stream().cuda_stream
    torch.cuda.synchronize()
    lib, p, st, null = L.lib(), lambda t: C.c_void_p(t.data_ptr()), C.c_void_p(stream), C.c_void_p(0)
    codes, args = [], [(p(q), p(s), p(w), p(ws), p(c[0])), (p(x), p(w), p(ws), p(c[1]))]
    calls = [lambda: codes.append(lib.ftm_fp8_gemm(moe._h, *args[0][:4], m, n, k, args[0][4], L.F32, n, st))]
    if m <= 16:
        calls.append(lambda: codes.append(lib.ftm_fp8_linear(moe._h, args[1][0], L.BF16, k, args[1][1], args[1][2], m, n, k, null, null, args[1][3], L.F32, n, st)))
    for call in calls:
        t = threading.Thread(target=call)
        t.start()
        t.join()
    torch.cuda.synchronize()
    assert codes == [L.OK] * len(calls)
    for i in range(len(calls)):
        assert torch.equal(c[i], want)


@pytest.mark.parametrize("out", ["bf16", "f32"])
@pytest.mark.parametrize("m,n,k", [(33, 300, 1040), (65, 257, 2048), (40, 9001, 1040), (60, 4099, 4112), (65, 2050, 8192), (100, 1000, 8192), (90, 8191, 2064),
                                   (100, 4097, 4112), (130, 2051, 8208), (500, 2000, 4112), (300, 4100, 400), (250, 4100, 1040)])
def test_tiles_of_every_width_whole_and_split(moe, m, n, k, out):
    """Tiles of 32, 64 and 128 tokens, each with a CTA of its own and with several that share its blocks."""
    q, s = moe.fp8_quantize(activations(m + n, m, k, torch.float32))
    w, ws = weight(k + n, n, k)
    buf = torch.full((m + 1, n + 3), 77.0, dtype=DT[out], device=DEV)
    c = buf[:m, :n]
    moe.fp8_gemm(q, s, w, ws, c)
    check_product(c, q.double().cpu().numpy(), s.cpu().numpy(), w, ws)
    assert (buf[:, n:] == 77.0).all() and (buf[m] == 77.0).all()
    again = torch.empty((m, n), dtype=DT[out], device=DEV)
    moe.fp8_gemm(q, s, w, ws, again)
    assert torch.equal(again, c)
    moe.sync_status()


@pytest.mark.parametrize("out", ["bf16", "f32"])
@pytest.mark.parametrize("n,ld,offset", [(1281, 1281, 0), (1407, 1407, 1), (1409, 1411, 0), (1534, 1534, 0), (1535, 1537, 3), (1539, 1540, 2), (1343, 1346, 0), (1280, 1284, 4),
                                         (1300, 1304, 8)])
def test_rows_of_pairs_start_and_end_anywhere(moe, n, ld, offset, out):
    m, k = 1100, 640
    q, s = moe.fp8_quantize(activations(n, m, k, torch.bfloat16))
    w, ws = weight(ld, n, k)
    buf = torch.full((m * ld + offset + 9,), 77.0, dtype=DT[out], device=DEV)
    c = buf.as_strided((m, n), (ld, 1), storage_offset=offset)
    moe.set_sm_budget(10)
    try:
        moe.fp8_gemm(q, s, w, ws, c)
        check_product(c, q.double().cpu().numpy(), s.cpu().numpy(), w, ws)
        moe.sync_status()
    finally:
        moe.set_sm_budget(0)
    kept = torch.ones_like(buf, dtype=torch.bool)
    kept.as_strided((m, n), (ld, 1), storage_offset=offset).fill_(False)
    assert (buf[kept] == 77.0).all()


@pytest.mark.parametrize("m,n,k", [(1, 40000, 2304), (16, 40000, 2816), (1, 40000, 2944), (3, 38000, 3200), (16, 40000, 3456), (1, 40000, 3840), (2, 40000, 3968),
                                   (16, 38000, 5120), (1, 40000, 8176), (5, 40000, 8192), (2, 12800, 5120), (16, 12800, 5888), (1, 12800, 6656), (4, 9000, 6912),
                                   (16, 9000, 7680), (1, 9000, 8192)])
def test_one_kernel_with_many_blocks_to_a_cta(moe, m, n, k):
    """Codes that leave the weight's ring little room, up to an SM for one CTA; whole and split over clusters."""
    x = activations(m + k, m, k, torch.bfloat16).contiguous()
    w, ws = weight(n + k, n, k)
    two = torch.empty((m, n), device=DEV)
    moe.fp8_gemm(*moe.fp8_quantize(x), w, ws, two)
    lib, p, st, null = L.lib(), lambda t: C.c_void_p(t.data_ptr()), C.c_void_p(torch.cuda.current_stream().cuda_stream), C.c_void_p(0)
    for _ in range(20):
        c = torch.full((m + 1, n), 77.0, device=DEV)
        assert lib.ftm_fp8_linear(moe._h, p(x), L.BF16, k, p(w), p(ws), m, n, k, null, null, p(c), L.F32, n, st) == L.OK
        assert torch.equal(c[:m], two) and (c[m] == 77.0).all()
    at = (n // 128 - 2) * 128
    check_product(c[:m, at:], *quantised(x), w[at:], ws[at // 128:])
    moe.sync_status()


def test_memory_that_is_still_read_is_not_taken_for_another_stream(moe):
    """A tensor of the scratch's or an output's size that was given back while a kernel of the current stream has yet to read it."""
    m, n, k = 64, 256, 2048
    x, (w, ws) = activations(1, m, k, torch.bfloat16), weight(2, n, k)
    logits, ids = activations(3, 512, 300, torch.float32), torch.zeros(512, dtype=torch.int64, device=DEV)
    side = torch.cuda.Stream()
    want, c, lp = torch.empty((m, n), device=DEV), torch.empty((m, n), device=DEV), moe.logprobs(logits, ids, 4)
    moe.fp8_linear(x, w, ws, want)
    torch.cuda.synchronize()
    sizes = [m * k, k // 128 * m * 4, 512 * 4, 512 * 16]
    for given in (side, side.cuda_stream):
        tensors = [torch.full((s,), 0x5a, dtype=torch.uint8, device=DEV) for s in sizes for _ in range(4)]
        torch.cuda._sleep(50_000_000)
        read = [t.clone() for t in tensors]
        del tensors
        moe.fp8_linear(x, w, ws, c, stream=given)
        codes = moe.fp8_quantize(x, stream=given)
        out = moe.logprobs(logits, ids, 4, stream=given)
        torch.cuda.synchronize()
        assert all((t == 0x5a).all() for t in read)
        assert torch.equal(c, want) and codes[0].shape == (m, k)
        for a, b in zip(out, lp):
            assert torch.equal(a, b)


@pytest.mark.parametrize("sms", [0, 40])
def test_scratch_is_made_where_two_kernels_are_taken(moe, sms):
    """Given or not, the same kernels run: two where the library says that a size uses its scratch, else one."""
    moe.set_sm_budget(sms)
    try:
        for m, n, k in [(1, 300, 16), (1, 40000, 2048), (1, 40000, 2064), (1, 40000, 4096), (1, 2048, 4096), (2, 20000, 4080), (2, 1000, 8192), (1, 60000, 8176),
                        (3, 200, 2048), (10, 5000, 2048), (11, 5000, 2048), (16, 40000, 1280), (16, 40000, 1296), (16, 130, 1296), (13, 2048, 4096), (16, 64, 8192),
                        (1, 64, 8208), (17, 64, 16), (40, 300, 256), (1, 230000, 2560), (8, 230000, 2560)]:
            x, (w, ws) = activations(m, m, k, torch.bfloat16).contiguous(), weight(k, n, k)
            scratch = moe.fp8_quantize(x)
            c = torch.empty((2, m, n), device=DEV)
            two = L.lib().ftm_fp8_linear_scratch(moe._h, m, n, k)
            assert two in (0, 1) and (two == 1 or (m <= 16 and k <= 8192))
            for i, given in enumerate((None, scratch)):
                before = moe.kernel_launches()
                moe.fp8_linear(x, w, ws, c[i], scratch=given)
                assert moe.kernel_launches() - before == 1 + two, (m, n, k, given is None)
            assert torch.equal(c[0], c[1])
        for sizes in ((0, 1, 16), (1, 0, 16), (1, 1, 0), (-1, 5, 16)):
            assert L.lib().ftm_fp8_linear_scratch(moe._h, *sizes) == 0
        moe.sync_status()
    finally:
        moe.set_sm_budget(0)


def test_scratch_of_sizes_that_are_refused(moe):
    ask = lambda m, n, k: L.lib().ftm_fp8_linear_scratch(moe._h, m, n, k)
    assert ask(17, 2 ** 30, 16) == 1 and ask(1, 64, 8208) == 1
    for sizes in ((17, 2 ** 31 - 1, 16), (1, 2 ** 31 - 1, 8192), (1, 2 ** 30 + 1, 8192), (2 ** 30 + 1, 1, 16), (17, 64, 2 ** 30 + 16), (17, 64, 24), (17, 64, 8)):
        assert ask(*sizes) == 0, sizes
    assert L.lib().ftm_fp8_linear_scratch(C.c_void_p(0), 17, 64, 16) == 0
