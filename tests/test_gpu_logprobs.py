"""Log probabilities of given tokens, ranks, entropies and the most probable alternatives, against the definition in 64 bits."""
import ctypes as C
import importlib

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
pkg = importlib.import_module("ferrum-torrens_b200")
L = pkg._lib

DT = {"bf16": torch.bfloat16, "f32": torch.float32}
DEV = "cuda:0"
INF = float("inf")


@pytest.fixture(scope="module")
def moe():
    m = pkg.B200MoE(0, pkg.ExpertShapes(64, 16), 1, experts=1, layers=1, top_k=1, shared_inter=16, max_tokens=1)
    yield m
    m.close()


def logits_of(seed, rows, vocab, dtype, pad=0, offset=0, spread=3.0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn((rows, vocab + pad), generator=gen, device=DEV) * spread).to(dtype)[:, offset:offset + vocab]


def definition(x, ids, n):
    """(logprob, entropy, rank, top ids, top logprobs) of one batch, and what the two kinds of values may be off by."""
    x = x.double().cpu().numpy()
    rows, vocab = x.shape
    order_by = np.where(np.isnan(x), -INF, x)
    lp, ent, rank = np.zeros(rows), np.zeros(rows), np.full(rows, -1)
    top, top_lp = np.full((rows, n), -1), np.full((rows, n), -INF)
    tol, tol_ent = np.zeros(rows), np.zeros(rows)
    for r in range(rows):
        v = x[r]
        order = np.argsort(-order_by[r], kind="stable")
        broken, empty = np.isnan(v).any() or (v == INF).any(), (v == -INF).all()
        if broken:
            logp = np.full(vocab, np.nan)
            ent[r] = np.nan
        elif empty:
            logp = np.full(vocab, -INF)
        else:
            m = v.max()
            e = np.exp(v - m)
            s = e.sum()
            logp = (v - m) - np.log(s)
            p = e / s
            live = p > 0
            dist = (p[live] * np.abs(v[live] - m)).sum()
            ent[r] = np.log(s) + dist
            # s: up to vocab / 256 + 40 additions in a chain, each half a step; exponentials within 2^-21 of the value, their
            # arguments off by their own size times 2^-23.  Then the logarithm, the differences and the result's rounding.
            rel = (vocab / 256 + 40) * 2.0 ** -24 + 2.0 ** -21 + dist * 2.0 ** -22
            tol[r] = rel + 2.0 ** -22 * (1 + np.log(s))
            tol_ent[r] = rel * (1 + 2 * dist) + 2.0 ** -22 * (1 + np.log(s) + dist)
        k = min(n, vocab)
        top[r, :k], top_lp[r, :k] = order[:k], logp[order[:k]]
        if 0 <= ids[r] < vocab:
            lp[r], rank[r] = logp[ids[r]], int(np.flatnonzero(order == ids[r])[0])
        elif ids[r] >= vocab:
            lp[r] = np.nan
    return (lp, ent, rank, top, top_lp), tol, tol_ent


def close(got, want, tol):
    got = got.double().cpu().numpy()
    same = np.isnan(want) == np.isnan(got)
    assert same.all()
    assert np.array_equal(got[np.isinf(want)], want[np.isinf(want)])
    f = np.isfinite(want)
    tol = np.broadcast_to(tol.reshape(tol.shape + (1,) * (want.ndim - 1)), want.shape) + np.where(f, np.abs(np.where(f, want, 0)), 0) * 2.0 ** -23
    d = np.abs(got[f] - want[f])
    assert (d <= tol[f]).all(), float((d / tol[f]).max())


def check(moe, x, ids, n, ids_dtype=torch.int64):
    got = moe.logprobs(x, ids.to(ids_dtype), n)
    want, tol, tol_ent = definition(x, ids.cpu().numpy(), n)
    assert np.array_equal(got[3].cpu().numpy(), want[3])
    assert np.array_equal(got[2].cpu().numpy(), want[2])
    close(got[0], want[0], tol)
    close(got[1], want[1], tol_ent)
    close(got[4], want[4], tol)
    again = moe.logprobs(x, ids.to(ids_dtype), n)
    for a, b in zip(got, again):
        assert torch.equal(a.view(torch.int32), b.view(torch.int32)), "the same inputs give the same bits"
    return got


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,vocab,n,pad,offset", [
    (1, 1, 1, 0, 0), (2, 2, 5, 0, 0), (3, 7, 7, 2, 1), (3, 31, 32, 0, 0), (1, 33, 20, 0, 0), (5, 1000, 0, 0, 0), (5, 1000, 1, 3, 2), (2, 4097, 20, 0, 0),
    (1, 40000, 32, 0, 0), (300, 513, 5, 0, 0), (3, 40001, 20, 7, 3), (700, 1500, 3, 0, 0), (1, 248320, 20, 0, 0), (2, 100003, 8, 0, 0), (9, 65536, 9, 64, 0),
    (40, 33000, 17, 1, 0), (650, 40001, 12, 0, 0), (800, 9000, 32, 5, 1), (13, 248320, 20, 0, 0), (150, 70000, 2, 0, 0)])
def test_random_rows(moe, rows, vocab, n, pad, offset, dtype):
    x = logits_of(rows + vocab, rows, vocab, DT[dtype], pad, offset)
    gen = torch.Generator(device=DEV).manual_seed(vocab)
    ids = torch.randint(0, vocab, (rows,), generator=gen, device=DEV)
    ids[::3] = x.float().argmax(-1)[::3]                 # likely tokens among them
    if rows > 4:
        ids[1], ids[2], ids[3] = -1, 0, vocab - 1
    check(moe, x, ids, n, torch.int32 if vocab % 2 else torch.int64)
    moe.sync_status()


def special_rows(vocab):
    g = torch.Generator().manual_seed(vocab)
    rnd = lambda: torch.randn(vocab, generator=g) * 3
    rows = []
    rows.append(torch.full((vocab,), -INF))                                # nothing left
    r = torch.full((vocab,), -INF); r[vocab // 2] = -3.0; rows.append(r)   # one left
    r = torch.full((vocab,), -INF); r[vocab // 3::max(1, vocab // 7)] = rnd()[vocab // 3::max(1, vocab // 7)]; rows.append(r)
    rows.append(torch.zeros(vocab))                                        # all equal
    r = torch.zeros(vocab); r[::2] = -0.0; rows.append(r)                  # the two zeros are equal
    low = torch.finfo(torch.bfloat16).min
    rows.append(torch.full((vocab,), low))                                 # masked by the lowest value throughout
    r = torch.full((vocab,), low); r[-1] = 1.0; rows.append(r)
    r = rnd(); r[torch.rand(vocab, generator=g) < 0.9] = low; rows.append(r)
    r = rnd(); r[torch.rand(vocab, generator=g) < 0.9] = -INF; rows.append(r)
    rows.append(torch.arange(vocab).float() * 0.01)                        # every element a new maximum
    rows.append(-torch.arange(vocab).float() * 0.01)
    rows.append((rnd() * 2).round())                                       # ties everywhere
    r = rnd(); r[vocab // 2] = 80.0; rows.append(r)                        # all but certain
    r = rnd(); r[vocab // 2] = INF; rows.append(r)
    r = rnd(); r[vocab - 1] = float("nan"); rows.append(r)
    rows.append(torch.full((vocab,), float("nan")))
    r = torch.full((vocab,), -INF); r[0] = float("nan"); rows.append(r)
    rows.append(torch.full((vocab,), INF))
    rows.append(rnd() * 1e37)                                              # differences that overflow
    rows.append(rnd() + 5e4)                                               # far from zero
    return torch.stack(rows)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("vocab,n", [(3, 5), (37, 32), (1001, 20), (9000, 32), (70001, 7)])
def test_special_rows(moe, vocab, n, dtype):
    x = special_rows(vocab).to(DT[dtype]).to(DEV)
    for at in (0, vocab // 2, vocab - 1, vocab // 3):
        check(moe, x, torch.full((x.shape[0],), at, device=DEV), n)
    # one row at a time: the split over a cluster
    for r in range(x.shape[0]):
        check(moe, x[r:r + 1], torch.full((1,), vocab // 2, device=DEV), n)
    moe.sync_status()


@pytest.mark.parametrize("vocab", [5, 5000, 100000])
def test_ids_outside_the_vocabulary(moe, vocab):
    x = logits_of(1, 6, vocab, torch.float32)
    ids = torch.tensor([0, -1, -100, vocab - 1, -2 ** 40, 3], device=DEV)
    check(moe, x, ids, 3)
    moe.sync_status()
    for wrong in (vocab, 2 ** 31 + 1, 2 ** 33):
        check(moe, x, torch.tensor([0, 1, wrong, 2, 3, 4], device=DEV), 3)
        with pytest.raises(pkg.MoEError, match="token id"):
            moe.sync_status()
        moe.sync_status()
    check(moe, x, torch.tensor([0, 1, vocab, -5, 3, 4], device=DEV), 3, torch.int32)
    with pytest.raises(pkg.MoEError, match="token id"):
        moe.sync_status()


def test_outputs_left_out_and_rows_behind_the_last(moe):
    rows, vocab, n = 7, 3000, 4
    x, ids = logits_of(2, rows, vocab, torch.bfloat16), torch.arange(rows, device=DEV)
    full = moe.logprobs(x, ids, n)
    lp, ent, rank, ti, tl = moe.logprobs(x, top_n=n)
    assert lp is None and rank is None and torch.equal(ent, full[1]) and torch.equal(ti, full[3]) and torch.equal(tl, full[4])
    for keep in range(5):
        bufs = [torch.full((rows + 2, *t.shape[1:]), 9, dtype=t.dtype, device=DEV) for t in full]
        out = [b[:rows] if i == keep or (keep >= 3 and i >= 3) else None for i, b in enumerate(bufs)]
        moe.logprobs(x, ids, n if keep >= 3 else 0, out=out)
        for i, (b, t) in enumerate(zip(bufs, full)):
            if out[i] is not None:
                assert torch.equal(b[:rows], t)
            assert (b[rows:] == 9).all()


def test_rows_past_32_bits(moe):
    rows, vocab, stride = 9, 5000, 2 ** 28 + 3
    buf = torch.empty((8 * stride + vocab,), dtype=torch.bfloat16, device=DEV)
    x = buf.as_strided((rows, vocab), (stride, 1))
    x.copy_(logits_of(3, rows, vocab, torch.bfloat16))
    check(moe, x, torch.arange(rows, device=DEV) * 500, 6)


def test_a_decode_tail_in_a_graph(moe):
    """Hidden rows -> projection to the vocabulary in 8 bits -> what is read off the logits: as calls, as a graph on new inputs, and on
    three streams at once."""
    m, k, vocab, n = 5, 512, 12000, 8
    gen = torch.Generator(device=DEV).manual_seed(4)
    w = (torch.randn((vocab, k), generator=gen, device=DEV) * 90).clamp(-448, 448).to(torch.float8_e4m3fn)
    ws = torch.full((-(-vocab // 128), k // 128), 1e-3, device=DEV)
    inputs = [torch.randn((m, k), generator=gen, device=DEV).bfloat16() for _ in range(3)]
    ids = torch.randint(0, vocab, (m,), generator=gen, device=DEV)

    def buffers():
        return (torch.empty((m, vocab), device=DEV), moe.fp8_quantize(inputs[0]),
                tuple(torch.empty(s, dtype=d, device=DEV) for s, d in (((m,), torch.float32), ((m,), torch.float32), ((m,), torch.int32), ((m, n), torch.int32), ((m, n), torch.float32))))

    def tail(x, logits, scratch, out):
        moe.fp8_linear(x, w, ws, logits, scratch=scratch)
        moe.logprobs(logits, ids, n, out=out)
        return out
    wanted = []
    for x in inputs:
        logits, scratch, out = buffers()
        tail(x, logits, scratch, out)
        want, tol, _ = definition(logits, ids.cpu().numpy(), n)
        assert np.array_equal(out[3].cpu().numpy(), want[3]) and np.array_equal(out[2].cpu().numpy(), want[2])
        close(out[0], want[0], tol)
        wanted.append(out)
    x = inputs[0].clone()
    logits, scratch, out = buffers()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        tail(x, logits, scratch, out)
    for i in (2, 1):
        x.copy_(inputs[i])
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, wanted[i]):
            assert torch.equal(a, b)
    streams, sets = [torch.cuda.Stream() for _ in range(3)], [buffers() for _ in range(3)]
    torch.cuda.synchronize()
    for _ in range(20):
        for st, x_in, b in zip(streams, inputs, sets):
            with torch.cuda.stream(st):
                tail(x_in, *b)
    torch.cuda.synchronize()
    for b, v in zip(sets, wanted):
        for t, u in zip(b[2], v):
            assert torch.equal(t, u)
    moe.sync_status()


def test_refusals(moe):
    x, ids = logits_of(0, 4, 100, torch.float32), torch.zeros(4, dtype=torch.int64, device=DEV)
    good = moe.logprobs(x, ids, 3)
    bad = [
        lambda: moe.logprobs(x.half(), ids), lambda: moe.logprobs(x.cpu(), ids), lambda: moe.logprobs(x[0], ids), lambda: moe.logprobs(x.t(), ids),
        lambda: moe.logprobs(x[:0], ids[:0]), lambda: moe.logprobs(x[:, :0], ids), lambda: moe.logprobs(x, ids[:3]), lambda: moe.logprobs(x, ids.float()),
        lambda: moe.logprobs(x, ids, 33), lambda: moe.logprobs(x, ids, -1), lambda: moe.logprobs(x, ids.cpu()), lambda: moe.logprobs(x, ids, 4, out=good),
        lambda: moe.logprobs(x, None, 3, out=good), lambda: moe.logprobs(x, ids, 3, out=(None, None, None, None, good[4])), lambda: moe.logprobs(x, ids, 0, out=(None,) * 5),
        lambda: moe.logprobs(x[:1].expand(4, 100), ids),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(pkg.MoEError) as e:
            call()
        assert e.value.kind == "Bad", i
    lib, null = L.lib(), C.c_void_p(0)
    p = lambda t, off=0: C.c_void_p(t.data_ptr() + off)
    run = lambda px=p(x), dt=L.F32, rows=4, vocab=100, ld=100, pi=p(ids), idt=L.I64, n=0, o=p(good[0]): lib.ftm_logprobs(
        moe._h, px, dt, rows, vocab, ld, pi, idt, n, o, null, null, null, null, null)
    assert run() == L.OK
    for kw in (dict(px=null), dict(dt=L.I32), dict(rows=0), dict(vocab=0), dict(vocab=2 ** 30 + 1, ld=2 ** 31), dict(ld=99), dict(pi=null), dict(idt=L.F32), dict(n=33),
               dict(n=2), dict(o=null), dict(px=p(x, 2)), dict(pi=p(ids, 4)), dict(o=p(good[0], 1))):
        assert run(**kw) == L.ERR_BAD, kw
    assert lib.ftm_logprobs(null, null, 0, 1, 1, 1, null, 2, 0, null, null, null, null, null, null) == L.ERR_BAD
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("vocab,n", [(5000, 5), (40001, 32), (248320, 20)])
def test_zeros_of_either_sign_far_apart(moe, vocab, n, dtype):
    """The two zeros are equal wherever they lie: stretches of one sign that are longer than what any warp reads at a time."""
    x = torch.zeros((4, vocab), device=DEV, dtype=DT[dtype])
    x[0, :vocab // 2] = -0.0
    x[1, vocab // 2:] = -0.0
    x[2, :vocab - 40] = -0.0
    x[3, 40:] = -0.0
    check(moe, x, torch.tensor([vocab // 3, vocab - 1, vocab - 5, 41], device=DEV), n)
    check(moe, x.repeat(160, 1), torch.tensor([vocab // 3, vocab - 1, vocab - 5, 41], device=DEV).repeat(160), n)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,vocab,n", [(1, 248320, 20), (3, 40001, 32), (640, 20003, 7), (160, 60000, 20)])
def test_more_ties_than_candidates(moe, rows, vocab, n, dtype):
    """Many elements that reach the bound, some tied with it and some above, in stretches, spread out and behind one another."""
    gen = torch.Generator(device=DEV).manual_seed(rows + vocab)
    x = torch.full((rows, vocab), torch.finfo(torch.bfloat16).min, device=DEV)
    steps = torch.arange(vocab, device=DEV)
    for r in range(min(rows, 160)):
        kind = r % 8 if rows > 3 else r + 3
        if kind == 1:
            x[r, 997::vocab // 5] = 1.0                  # fewer left than alternatives
        elif kind == 2:
            x[r, vocab // 3:] = 2.0
        elif kind == 3:
            x[r] = (torch.rand(vocab, generator=gen, device=DEV) * 5).floor()
        elif kind == 4:
            x[r] = (steps * 64 // vocab).float()
        elif kind == 5:
            x[r] = -(steps * 64 // vocab).float()
            x[r, -3:] = 1.0
        elif kind == 6:
            x[r, -700:] = 3.0
            x[r, -1] = 4.0
            x[r, ::211] = 3.0
        elif kind == 7:
            x[r] = float("nan")
            x[r, 5::2] = 1.0
    x[160:] = x[:160].repeat(4, 1)[:max(0, rows - 160)]
    ids = torch.randint(0, vocab, (rows,), generator=gen, device=DEV)
    x = x.to(DT[dtype])
    got = moe.logprobs(x, ids, n)
    if rows > 160:
        for t in (got[1], got[3], got[4]):               # (their tokens differ)
            for i in range(160, rows, 160):
                assert torch.equal(t[i:i + 160].view(torch.int32), t[:160].view(torch.int32))
    x, ids = x[:160], ids[:160]
    want, _, _ = definition(x, ids.cpu().numpy(), n)
    assert np.array_equal(got[3][:160].cpu().numpy(), want[3]) and np.array_equal(got[2][:160].cpu().numpy(), want[2])
    check(moe, x, ids, n)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,vocab", [(3, 700), (700, 1500), (5, 40001), (1, 248320), (300, 70000)])
def test_tokens_that_are_all_but_certain(moe, rows, vocab, dtype):
    """The log probability of such a token, and its row's entropy, to the precision of their own small values."""
    x = logits_of(rows, rows, vocab, DT[dtype])
    x = x.clamp(max=14)
    gen = torch.Generator(device=DEV).manual_seed(vocab)
    ids = torch.randint(0, vocab, (rows,), generator=gen, device=DEV)
    ids[0] = vocab - 1
    x[torch.arange(rows, device=DEV), ids] = torch.tensor([22.0, 28.0, 20.0, 34.0, 25.0], device=DEV).repeat(rows)[:rows].to(DT[dtype])
    got = moe.logprobs(x, ids, 1)
    d = x.double() - x.double().amax(-1, keepdim=True)
    e = d.exp()
    e[torch.arange(rows, device=DEV), ids] = 0.0
    rest = e.sum(-1)
    dist = -(e * torch.where(e > 0, d, 0.0)).sum(-1)
    lp, ent = -torch.log1p(rest), torch.log1p(rest) + dist / (1 + rest)
    # of the rest's sum: vocab / 256 + 40 additions, exponentials within 2^-21, their arguments (up to 60) off by their own size times 2^-23
    tol = (vocab / 256 + 40) * 2.0 ** -24 + 2.0 ** -21 + 60 * 2.0 ** -22
    assert ((got[0].double() - lp).abs() <= tol * lp.abs()).all()
    assert torch.equal(got[4][:, 0], got[0])
    assert ((got[1].double() - ent).abs() <= 2 * tol * ent).all()
    assert (got[2] == 0).all() and torch.equal(got[3][:, 0].long(), ids)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_the_largest_vocabularies(moe, dtype):
    """Parts of more tiles than there are notes: one row of 2^24, and rows of 600001 that have a CTA each."""
    x = logits_of(1, 1, 2 ** 24, DT[dtype])
    check(moe, x, torch.tensor([2 ** 24 - 5], device=DEV), 32)
    x[0, 5::1000] = 30.0                                 # more ties than candidates
    check(moe, x, torch.tensor([2 ** 23 + 5], device=DEV), 20)
    del x
    rows, vocab, n = 650, 600001, 20
    x = logits_of(2, rows, vocab, DT[dtype])
    x[1, ::3] = 20.0
    x[2] = torch.arange(vocab, device=DEV).float() / 1024
    ids = torch.randint(0, vocab, (rows,), generator=torch.Generator(device=DEV).manual_seed(1), device=DEV)
    got = moe.logprobs(x, ids, n)
    some = [0, 1, 2, 300, rows - 1]
    want, tol, tol_ent = definition(x[some], ids[some].cpu().numpy(), n)
    assert np.array_equal(got[3][some].cpu().numpy(), want[3]) and np.array_equal(got[2][some].cpu().numpy(), want[2])
    close(got[0][some], want[0], tol)
    close(got[1][some], want[1], tol_ent)
    close(got[4][some], want[4], tol)
    moe.sync_status()


FAR = [s * m for m in (3.9e6, 4.1e6, 1e8, 3e9, 5e9, 1e10, 1e12, 1e20, 9e29) for s in (1.0, -1.0)]


def far_rows(vocab):
    """Finite rows whose maxima lie anywhere between the usual logits and the type's limits, and masks of such values."""
    g = torch.Generator().manual_seed(vocab)
    rnd = lambda: torch.randn(vocab, generator=g) * 3
    rows = []
    for far in FAR:
        rows.append(torch.full((vocab,), far))
        rows.append(rnd() + far)                                           # as close as the type's steps are there
        rows.append(far + abs(far) * 0.1 * rnd())
        if far > 0:
            r = rnd(); r[vocab // 3] = far; rows.append(r)                 # the maximum rises to it
        else:
            r = rnd(); r[torch.rand(vocab, generator=g) < 0.9] = far; rows.append(r)
            r = torch.full((vocab,), far); r[-3:] = rnd()[-3:]; rows.append(r)         # first tiles with nothing else
            r = torch.full((vocab,), far); r[::2] = -INF; r[vocab // 2] = far * 0.5; rows.append(r)
    return torch.stack(rows)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("vocab,n,times", [(37, 5, 1), (700, 3, 10), (9000, 20, 9), (70001, 20, 1), (70001, 5, 9)])
def test_rows_far_from_zero(moe, vocab, n, times, dtype):
    """Whole rows and, with `times` of each, rows enough for a CTA of eight or of four warps each."""
    x = far_rows(vocab).to(DT[dtype]).to(DEV)
    ids = torch.randint(0, vocab, (x.shape[0],), generator=torch.Generator().manual_seed(n)).to(DEV)
    ids[::2] = x.float().argmax(-1)[::2]
    want, tol, tol_ent = definition(x, ids.cpu().numpy(), n)
    # x log2(e) - c is held in f32 where |x| < 4e6, with |c - x log2(e)| < 0.75: within the arguments' 2^-23 and the exponentials' 2^-21
    tile = lambda v: np.tile(v, (times,) + (1,) * (v.ndim - 1))
    got = moe.logprobs(x.repeat(times, 1), ids.repeat(times), n)
    assert np.array_equal(got[3].cpu().numpy(), tile(want[3])) and np.array_equal(got[2].cpu().numpy(), tile(want[2]))
    close(got[0], tile(want[0]), tile(tol))
    close(got[1], tile(want[1]), tile(tol_ent))
    close(got[4], tile(want[4]), tile(tol))
    if times == 1:
        for r in range(x.shape[0]):
            check(moe, x[r:r + 1], ids[r:r + 1], n)
    moe.sync_status()
