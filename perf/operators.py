"""The dense operators of the decode tail whose speed is kept track of: the 8-bit projection and what is read off its logits.

Four operators, in a plain form made of elementary torch operations and, where `own` is set, through the adapter's calls:

* "quantize": `fp8_quantize`, activation rows to e4m3 with one scale for each row and block of 128 elements.
* "gemm": `fp8_gemm`, quantised rows times a weight of e4m3 with one scale for each block of 128 x 128, as checkpoints in
  8 bits hold them.
* "linear": `fp8_linear`, the same product on rows that are still bf16 or f32: a decode step's call.
* "logprobs": `logprobs`, from rows of logits the given tokens' log probabilities and ranks, the rows' entropies and the
  most probable alternatives; `masked` = the share of the vocabulary that a grammar rules out (-inf; with more than four rows one
  row is ruled out whole), `unasked` = rows at the end of the batch without a token, `pad` = columns of the buffer behind
  the vocabulary.

Every input is drawn from the seed, on the GPU.  The outputs are buffers that the caller owns, as in a decode loop.
"""
import importlib

import torch

own = False

HIDDEN, VOCAB, BLOCK = 2048, 248320, 128
E4M3_MAX, SMALLEST = 448.0, 2.0 ** -126
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32, "i32": torch.int32, "i64": torch.int64}
SIZE = {"bf16": 2, "f32": 4}
MOST_FLOPS = 2 * 8192 * 8192 * 4096
MOST_WEIGHT = VOCAB * HIDDEN
MOST_LOGITS = 999 * VOCAB


def _quantize(name, rows, k, x="bf16"):
    return {"name": name, "op": "quantize", "rows": rows, "k": k, "x": x}


def _gemm(name, m, n, k, out="bf16"):
    return {"name": name, "op": "gemm", "m": m, "n": n, "k": k, "out": out}


def _linear(name, m, n, k, x="bf16", out="bf16"):
    return {"name": name, "op": "linear", "m": m, "n": n, "k": k, "x": x, "out": out}


def _logprobs(name, rows, vocab, top, x="f32", ids="i64", masked=0.0, unasked=0, pad=0):
    return {"name": name, "op": "logprobs", "rows": rows, "vocab": vocab, "top": top, "x": x, "ids": ids, "masked": masked,
            "unasked": unasked, "pad": pad}


def listed():
    return [
        # the hidden rows of a decode batch: latency
        _quantize("quantize-37", 37, HIDDEN),
        # a chunk of many prompts at twice the hidden size (the input of an output projection)
        _quantize("quantize-8192", 8192, 2 * HIDDEN),
        # one sequence being decoded: an input projection
        _linear("linear-1", 1, 8192, HIDDEN),
        # a ragged decode batch: an output projection, few weight rows and a long sum, everything in f32
        _linear("linear-13-f32", 13, HIDDEN, 2 * HIDDEN, x="f32", out="f32"),
        # the vocabulary projection of eight sequences, logits in f32
        _linear("linear-8-vocab", 8, VOCAB, HIDDEN, out="f32"),
        # a decode batch whose rows were quantised once for several projections
        _gemm("gemm-64", 64, 10240, HIDDEN),
        # a ragged prompt on a weight whose sizes are no multiple of the scales' block
        _gemm("gemm-1000-ragged", 1000, 4100, 2000),
        # the largest: a batch of prompts
        _gemm("gemm-8192", 8192, 8192, 2 * HIDDEN),
        # the token just sampled by one sequence, with as many alternatives as servers offer
        _logprobs("logprobs-1", 1, VOCAB, 20),
        # a decode batch under a grammar, some of its rows idle, in a buffer wider than the vocabulary
        _logprobs("logprobs-64-masked", 64, VOCAB, 5, masked=0.9, unasked=3, pad=64),
        # the log probabilities of a prompt, logits in bf16
        _logprobs("logprobs-999-bf16", 999, VOCAB, 1, x="bf16", ids="i32"),
        # many prompts over a small vocabulary of odd size: no row but the first starts on a 16-byte boundary
        _logprobs("logprobs-4096-odd", 4096, 32003, 20, x="bf16"),
    ]


def _log_int(rng, lo, hi):
    """An integer of [lo, hi], uniform in its logarithm."""
    return min(hi, max(lo, int(lo * (hi / lo) ** rng.random() + 0.5)))


def _log_16(rng, lo, hi):
    return 16 * _log_int(rng, lo // 16, hi // 16)


def draw(rng):
    op = rng.choice(["quantize", "gemm", "gemm", "linear", "linear", "logprobs", "logprobs"])
    if op == "quantize":
        k = _log_16(rng, 128, 8192)
        return {"op": op, "rows": _log_int(rng, 1, 8192 * 2 * HIDDEN // max(k, 2 * HIDDEN)), "k": k, "x": rng.choice(["bf16", "bf16", "f32"])}
    if op == "gemm":
        n, k = _log_int(rng, 64, 16384), _log_16(rng, 128, 8192)
        return {"op": op, "m": _log_int(rng, 1, min(8192, MOST_FLOPS // (2 * n * k))), "n": n, "k": k, "out": rng.choice(["bf16", "bf16", "f32"])}
    if op == "linear":
        k = _log_16(rng, 128, 8192)
        return {"op": op, "m": _log_int(rng, 1, 64), "n": _log_int(rng, 64, min(VOCAB, MOST_WEIGHT // k)), "k": k,
                "x": rng.choice(["bf16", "bf16", "f32"]), "out": rng.choice(["bf16", "f32"])}
    rows = _log_int(rng, 1, 4096)
    return {"op": op, "rows": rows, "vocab": _log_int(rng, 1000, min(VOCAB, MOST_LOGITS // rows)), "top": rng.randint(1, 32),
            "x": rng.choice(["bf16", "f32"]), "ids": rng.choice(["i32", "i64"]), "masked": rng.choice([0.0, 0.0, 0.5, 0.99]),
            "unasked": rows // 8 if rng.random() < 0.3 else 0, "pad": rng.choice([0, 0, 5, 64])}


def _activations(gen, rows, k):
    """Rows as they leave a norm: about unit scale, a scale of its own for each row and a few columns far above the rest."""
    x = torch.randn((rows, k), generator=gen, device="cuda")
    x *= torch.exp2(torch.randn((rows, 1), generator=gen, device="cuda"))
    loud = torch.randint(0, k, (max(1, k // 512),), generator=gen, device="cuda")
    x[:, loud] *= 12.0
    return x


def _weight(gen, n, k):
    """A weight as an 8-bit checkpoint holds it: e4m3 codes that use the type's range, block scales around 1e-4."""
    w = torch.empty((n, k), dtype=torch.float8_e4m3fn, device="cuda")
    for i in range(0, n, 32768):
        w[i:i + 32768] = (torch.randn((min(32768, n - i), k), generator=gen, device="cuda") * 100.0).clamp_(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    scale = 2e-4 * torch.exp2(torch.randn((-(-n // BLOCK), -(-k // BLOCK)), generator=gen, device="cuda") * 0.5)
    return w, scale


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s, op = {"op": case["op"]}, case["op"]
    if op == "logprobs":
        rows, vocab, top, asked = case["rows"], case["vocab"], case["top"], case["rows"] - case["unasked"]
        x = torch.randn((rows, vocab + case["pad"]), generator=gen, device="cuda") * 2.5
        ids = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
        # the given token stands out, more or less: sampled tokens are mostly likely ones
        x[torch.arange(rows, device="cuda"), ids] += 9.0 + 3.0 * torch.randn(rows, generator=gen, device="cuda")
        if case["masked"]:
            for i in range(0, rows, 256):
                out = torch.rand((min(256, rows - i), vocab + case["pad"]), generator=gen, device="cuda") < case["masked"]
                x[i:i + 256].masked_fill_(out, float("-inf"))
            x[torch.arange(rows, device="cuda"), ids] = 8.0
            if rows > 4:
                x[rows // 2] = float("-inf")
        ids[asked:] = -1
        s["logits"], s["ids"], s["top"] = x.to(DTYPES[case["x"]])[:, :vocab], ids.to(DTYPES[case["ids"]]), top
        new = lambda dtype, *shape: torch.empty(shape, dtype=dtype, device="cuda")
        s["out"] = (new(torch.float32, rows), new(torch.float32, rows), new(torch.int32, rows), new(torch.int32, rows, top), new(torch.float32, rows, top))
        return s
    if op == "quantize":
        rows, k = case["rows"], case["k"]
        s["x"] = _activations(gen, rows, k).to(DTYPES[case["x"]])
        s["out"] = (torch.empty((rows, k), dtype=torch.float8_e4m3fn, device="cuda"), torch.empty((-(-k // BLOCK), rows), dtype=torch.float32, device="cuda"))
        return s
    m, n, k = case["m"], case["n"], case["k"]
    s["w"], s["w_scale"] = _weight(gen, n, k)
    s["out"] = torch.empty((m, n), dtype=DTYPES[case["out"]], device="cuda")
    x = _activations(gen, m, k)
    if op == "gemm":
        s["a"], s["a_scale"] = _quantized(x)
    else:
        s["x"] = x.to(DTYPES[case["x"]])
        s["scratch"] = (torch.empty((m, k), dtype=torch.float8_e4m3fn, device="cuda"), torch.empty((-(-k // BLOCK), m), dtype=torch.float32, device="cuda"))
    return s


def _blocks(x):
    """[rows, k] as [rows, blocks, 128], the last block filled up with zeros."""
    rows, k = x.shape
    return torch.nn.functional.pad(x, (0, -k % BLOCK)).reshape(rows, -1, BLOCK)


def _quantized(x):
    """Codes [rows, k] and scales [blocks, rows] of rows in f32: the block's largest magnitude becomes 448."""
    xb = _blocks(x)
    most = xb.abs().amax(-1, keepdim=True).clamp(min=E4M3_MAX * SMALLEST)
    full = torch.full_like(most, E4M3_MAX)        # quotients of tensors: with a number torch multiplies by a rounded reciprocal
    q = (xb * (full / most)).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    return q.reshape(x.shape[0], -1)[:, :x.shape[1]].contiguous(), (most / full)[..., 0].t().contiguous()


def _product(a, a_scale, w, w_scale):
    """The product in f32: both operands as the values they stand for."""
    k = a.shape[1]
    rows = a.float() * a_scale.t().repeat_interleave(BLOCK, 1)[:, :k]
    cols = w.float() * w_scale.repeat_interleave(BLOCK, 1)[:, :k].repeat_interleave(BLOCK, 0)[:w.shape[0]]
    return rows @ cols.t()


def _read_off(logits, ids, top):
    x = logits.float() + 0.0          # -0 becomes 0: the two are one value and go by their index
    rows, vocab = x.shape
    m = x.amax(-1, keepdim=True)
    empty = m == float("-inf")
    d = torch.where(empty, float("-inf"), x - m)
    e = d.exp()
    total = e.sum(-1, keepdim=True)
    log_total = torch.where(empty, 0.0, total.log())
    entropy = torch.where(empty, 0.0, log_total - torch.where(e > 0, e * d, 0.0).sum(-1, keepdim=True) / total)[:, 0]
    # one whole number for each (value, index), larger for larger values, for equal ones where the index is lower
    bits = x.view(torch.int32)
    order = (bits ^ ((bits >> 31) & 0x7fffffff)).to(torch.int64) * 2 ** 32 + (vocab - 1 - torch.arange(vocab, device=x.device))
    top_ids = vocab - 1 - (order.topk(top, -1).values & 0xffffffff)
    asked = ids >= 0
    at = ids.clamp(min=0).to(torch.int64)[:, None]
    logprob = torch.where(asked, (d.gather(1, at) - log_total)[:, 0], 0.0)
    rank = torch.where(asked, (order > order.gather(1, at)).sum(-1), -1)
    return logprob, entropy, rank.to(torch.int32), top_ids.to(torch.int32), d.gather(1, top_ids) - log_total


_adapter = None


def _moe():
    """The process's adapter, made by the first call."""
    global _adapter
    if _adapter is None:
        ft = importlib.import_module("ferrum-torrens_b200")
        _adapter = ft.B200MoE(0, ft.ExpertShapes(HIDDEN, 16), 1, experts=1, layers=1, top_k=1, shared_inter=0, max_tokens=1)
    return _adapter


def run(s):
    op = s["op"]
    if op == "quantize":
        if own:
            return _moe().fp8_quantize(s["x"], out=s["out"])
        return _quantized(s["x"].float())
    if op == "gemm":
        if own:
            return _moe().fp8_gemm(s["a"], s["a_scale"], s["w"], s["w_scale"], s["out"])
        return _product(s["a"], s["a_scale"], s["w"], s["w_scale"]).to(s["out"].dtype)
    if op == "linear":
        if own:
            return _moe().fp8_linear(s["x"], s["w"], s["w_scale"], s["out"], scratch=s["scratch"])
        return _product(*_quantized(s["x"].float()), s["w"], s["w_scale"]).to(s["out"].dtype)
    if own:
        return _moe().logprobs(s["logits"], s["ids"], s["top"], out=s["out"])
    return _read_off(s["logits"], s["ids"], s["top"])


def work(case):
    if case["op"] == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        return {"bytes": rows * (vocab * SIZE[case["x"]] + (4 if case["ids"] == "i32" else 8) + 12 + 8 * case["top"]), "flops": 8 * rows * vocab}
    if case["op"] == "quantize":
        rows, k = case["rows"], case["k"]
        return {"bytes": rows * (k * SIZE[case["x"]] + k + 4 * -(-k // BLOCK)), "flops": 3 * rows * k}
    m, n, k = case["m"], case["n"], case["k"]
    blocks = -(-k // BLOCK)
    rows = m * (k + 4 * blocks) if case["op"] == "gemm" else m * k * SIZE[case["x"]]
    return {"bytes": rows + n * k + 4 * -(-n // BLOCK) * blocks + m * n * SIZE[case["out"]], "flops": 2 * m * n * k}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "logprobs":
        lp, entropy, top = [], [], []
        for i in range(0, case["rows"], 128):
            x, ids = s["logits"][i:i + 128].double(), s["ids"][i:i + 128].long()
            total = torch.logsumexp(x, -1, keepdim=True)
            every = torch.where(total == float("-inf"), float("-inf"), x - total)
            p = every.exp()
            entropy.append(-(p * torch.where(p > 0, every, 0.0)).sum(-1))
            top.append(every.sort(-1, descending=True).values[:, :case["top"]].clone())
            lp.append(torch.where(ids >= 0, every.gather(1, ids.clamp(min=0)[:, None])[:, 0], 0.0))
        return torch.cat(lp), torch.cat(entropy), None, None, torch.cat(top)

    def codes(x):
        """The definition's two roundings to f32 (a quotient or product of f32 values in 64 bits rounds to f32 as the
        f32 operation does) and the one to e4m3: multiples of the value's own step, ties to even."""
        q, scales = torch.empty(x.shape, dtype=torch.float64, device=x.device), []
        for b in range(0, x.shape[1], BLOCK):
            v = x[:, b:b + BLOCK].double()
            most = v.abs().max(-1).values.clamp(min=448.0 * 2.0 ** -126)
            y = (v * (448.0 / most).float().double()[:, None]).float().double()
            step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
            q[:, b:b + BLOCK] = (torch.round(y / step) * step).clamp(-448.0, 448.0)
            scales.append((most / 448.0).float().double())
        return q, torch.stack(scales)

    if case["op"] == "quantize":
        return codes(s["x"])
    if case["op"] == "gemm":
        q, scales = s["a"].double(), s["a_scale"].double()
    else:
        q, scales = codes(s["x"])
    c = torch.zeros((case["m"], case["n"]), dtype=torch.float64, device="cuda")
    for b in range(scales.shape[0]):
        at = slice(b * BLOCK, (b + 1) * BLOCK)
        by = s["w_scale"][:, b].double().repeat_interleave(BLOCK)[:case["n"]]
        c += (q[:, at] * scales[b][:, None]) @ (s["w"][:, at].double() * by[:, None]).t()
    return c
