"""The 8-bit products and log probabilities refuse what no device call could take before the library is reached (CPU)."""
import importlib

import pytest

torch = pytest.importorskip("torch")
pkg = importlib.import_module("ferrum-torrens_b200")
E4M3 = torch.float8_e4m3fn


class NoLibrary:
    def __getattr__(self, name):
        raise AssertionError(f"{name} was reached")


@pytest.fixture()
def moe(monkeypatch):
    m = object.__new__(pkg.B200MoE)
    m._lib, m._h, m.device, m._own_stream = NoLibrary(), None, 0, 0
    monkeypatch.setattr(m, "_on", lambda stream: 0, raising=False)
    return m


def refused(call, words):
    with pytest.raises(pkg.MoEError, match=words) as e:
        call()
    assert e.value.kind == "Bad"


def test_host_tensors_types_and_shapes(moe):
    x, w, ws = torch.zeros((4, 256), dtype=torch.bfloat16), torch.zeros((130, 256), dtype=E4M3), torch.zeros((2, 2))
    c, q, s = torch.zeros((4, 130)), torch.zeros((4, 256), dtype=E4M3), torch.zeros((2, 4))
    refused(lambda: moe.fp8_quantize(x), "must be on device 0")
    refused(lambda: moe.fp8_quantize(x.half()), "cannot be torch.float16")
    refused(lambda: moe.fp8_gemm(q, s, w, ws, c), "must be on device 0")
    refused(lambda: moe.fp8_gemm(x, s, w[:, :128], ws, c), "a weight .N, K. is wanted")
    refused(lambda: moe.fp8_gemm(q[0], s, w, ws, c), "a weight .N, K. is wanted")
    refused(lambda: moe.fp8_linear(x, w.to(torch.uint8), ws, c), "must be on device 0")
    refused(lambda: moe.fp8_linear(x.to(torch.int32), w, ws, c), "cannot be torch.int32")
    refused(lambda: moe.logprobs(c, torch.zeros(4, dtype=torch.int64), 3), "must be on device 0")
    refused(lambda: moe.logprobs(c.double(), None), "cannot be torch.float64")


def test_reasons_name_what_is_wrong(moe, monkeypatch):
    monkeypatch.setattr(torch.Tensor, "get_device", lambda self: 0)
    x = torch.zeros((4, 256), dtype=torch.bfloat16)
    refused(lambda: moe.fp8_quantize(x[0]), "two dimensions")
    refused(lambda: moe.fp8_quantize(x.t()), "contiguous in its last dimension")
    w, ws, c = torch.zeros((130, 256), dtype=E4M3), torch.zeros((2, 2)), torch.zeros((4, 130))
    refused(lambda: moe.fp8_linear(x, w, torch.zeros((2, 3)), c), r"scales is \(2, 3\), expected \(2, 2\)")
    refused(lambda: moe.fp8_linear(x, w, ws, c[:, :129]), r"output is \(4, 129\), expected \(4, 130\)")
    refused(lambda: moe.fp8_linear(x, w, ws.t(), c), "must be contiguous")
    refused(lambda: moe.logprobs(c, torch.zeros(3, dtype=torch.int64)), r"token ids is \(3,\)")
    refused(lambda: moe.logprobs(c, torch.zeros(4)), "token ids cannot be torch.float32")
    refused(lambda: moe.logprobs(c, None, 33), "at most 32")


class Streams:
    """Stands in for CUDA's streams and the library: notes the stream that each tensor is made on and each that is told of it."""

    def __init__(self, monkeypatch, module):
        self.now, self.made, self.told = 5, [], []
        outer, empty = self, torch.empty

        class Stream:
            def __init__(self, handle, device=None):
                self.handle = handle

            def __enter__(self):
                self.before, outer.now = outer.now, self.handle

            def __exit__(self, *_):
                outer.now = self.before

        def noted(*a, **kw):
            outer.made.append(outer.now)
            return empty(*a, **kw)
        monkeypatch.setattr(module, "_current_stream", lambda: lambda ordinal: outer.now)
        monkeypatch.setattr(torch.cuda, "ExternalStream", Stream)
        monkeypatch.setattr(torch.cuda, "stream", lambda s: s)
        monkeypatch.setattr(torch.cuda, "default_stream", lambda device=None: Stream(0))
        monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: Stream(outer.now))
        monkeypatch.setattr(torch, "empty", noted)
        monkeypatch.setattr(torch.Tensor, "get_device", lambda self: 0)
        monkeypatch.setattr(torch.Tensor, "record_stream", lambda self, s: outer.told.append(s.handle))

    def __getattr__(self, name):
        return lambda *a: 0


@pytest.mark.parametrize("given,own,on", [(9, 0, 9), (0, 0, 0), (0, 7, 7), (5, 0, 5), (0, 5, 5)])
def test_what_a_call_makes_comes_from_the_stream_of_the_call(monkeypatch, given, own, on):
    """From the current stream's memory it could be a block that is still read there.  5 is the current stream, 0 the default one or the
    adapter's own."""
    x, w, ws, c = torch.zeros((20, 256)), torch.zeros((130, 256), dtype=E4M3), torch.zeros((2, 2)), torch.zeros((20, 130))
    ids = torch.zeros(20, dtype=torch.int64)
    m = object.__new__(pkg.B200MoE)
    streams = Streams(monkeypatch, importlib.import_module("ferrum-torrens_b200.moe"))
    m._lib, m._h, m.device, m._own_stream = streams, None, 0, own
    for call, tensors, kept in ((lambda: m.fp8_quantize(x, stream=given), 2, True), (lambda: m.fp8_linear(x, w, ws, c, stream=given), 1, False),
                                (lambda: m.logprobs(c, ids, 3, stream=given), 5, True), (lambda: m.logprobs(c, None, stream=given), 3, True)):
        streams.made.clear(), streams.told.clear()
        call()
        assert streams.made == [on] * tensors
        # what the caller gets may be in use on the current stream when it is dropped
        assert streams.told == ([5] * tensors if kept and on != 5 else [])


def test_sizes_past_32_bits_are_not_cut(moe, monkeypatch):
    """The library takes sizes of 32 bits: what is larger would arrive there as another size, perhaps a valid one."""
    monkeypatch.setattr(torch.Tensor, "get_device", lambda self: 0)
    new = lambda dtype, *shape: torch.empty(shape, dtype=dtype, device="meta")
    bf16, f32, i64, many = torch.bfloat16, torch.float32, torch.int64, 2 ** 32 + 16
    refused(lambda: moe.fp8_quantize(new(bf16, many, 16), out=(new(E4M3, many, 16), new(f32, 1, many))), "2.30")
    refused(lambda: moe.fp8_quantize(new(bf16, 2, many), out=(new(E4M3, 2, many), new(f32, many // 128 + 1, 2))), "2.30")
    w, ws = new(E4M3, 8, 16), new(f32, 1, 1)
    refused(lambda: moe.fp8_gemm(new(E4M3, many, 16), new(f32, 1, many), w, ws, new(f32, many, 8)), "2.30")
    refused(lambda: moe.fp8_linear(new(bf16, many, 16), w, ws, new(f32, many, 8)), "2.30")
    refused(lambda: moe.fp8_linear(new(bf16, 4, 16), new(E4M3, many, 16), new(f32, many // 128 + 1, 1), new(f32, 4, many)), "2.30")
    refused(lambda: moe.fp8_linear(new(bf16, 4, many), new(E4M3, 8, many), new(f32, 1, many // 128 + 1), new(f32, 4, 8)), "2.30")
    refused(lambda: moe.logprobs(new(bf16, many, 5), None), "2.24")
    refused(lambda: moe.logprobs(new(f32, 3, many), new(i64, 3), out=(new(f32, 3), None, None, None, None)), "2.24")
