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
