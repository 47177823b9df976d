"""Refusals of the 8-bit float Linear's entry points: raised on the host, before anything is launched (no GPU: handles are fakes that fail)."""
import pytest
import torch


@pytest.fixture
def ops(monkeypatch):
    import tfmq_dm_amd.ops as ops

    class Never:
        def call(self, name, *a):
            raise AssertionError(f"{name} was launched")
    monkeypatch.setattr(ops, "_dev", lambda t: 0)
    monkeypatch.setattr(ops, "_stream", lambda d: None)
    monkeypatch.setattr(ops, "_lib_handle", lambda d=0, p=0: Never())
    return ops


def _pw(ops, N=20, K=40):
    return ops.PackedFp8(torch.zeros(N, 128, dtype=torch.uint8), torch.zeros(K, 128, dtype=torch.uint8), torch.ones(1, 1), None, N, K)


def test_cpu_tensors_are_refused():
    import tfmq_dm_amd.ops as ops
    for f in (ops.quantize_fp8, ops.pack_w_fp8):
        with pytest.raises(ops.TfmqError, match="no CPU fallback"):
            f(torch.zeros(4, 4))


@pytest.mark.parametrize("x,why", [
    (torch.zeros(4, 40, dtype=torch.float64), "fp32, fp16 or bf16"),
    (torch.zeros(4, 40, dtype=torch.int32), "fp32, fp16 or bf16"),
    (torch.zeros(40, 4).t(), "unit stride"),
    (torch.zeros(4, 6, 40).transpose(0, 1), "collapse"),
    (torch.zeros(1, 40).expand(4, 40), "overlap"),
    (torch.zeros(4, 39), "39 channels"),
])
def test_linear_refuses(ops, x, why):
    with pytest.raises(ops.TfmqError, match=why):
        ops.linear_fp8(x, _pw(ops))


def test_other_refusals(ops):
    pw = _pw(ops)
    with pytest.raises(ops.TfmqError, match="output type"):
        ops.linear_fp8(torch.zeros(4, 40), pw, out_dtype=torch.int8)
    with pytest.raises(ops.TfmqError, match=r"\[N, K\]"):
        ops.pack_w_fp8(torch.zeros(4, 4, 4))
    with pytest.raises(ops.TfmqError, match="bias must be"):
        ops._bias_f32(torch.zeros(3), 20, 0, "x")
    with pytest.raises(ops.TfmqError, match="float8_e4m3fn"):
        ops.load_w_fp8(torch.zeros(4, 4), torch.ones(1, 1))
    with pytest.raises(ops.TfmqError, match="scale must be"):
        ops.load_w_fp8(torch.zeros(4, 4).to(torch.float8_e4m3fn), torch.ones(2, 1))
    with pytest.raises(ops.TfmqError, match="do not fit"):
        ops.linear_fp8_bwd(torch.zeros(4, 40), torch.zeros(5, 20), pw)
    with pytest.raises(ops.TfmqError, match="do not fit"):
        ops.linear_fp8_bwd(torch.zeros(4, 40), torch.zeros(4, 21), pw)


def test_operands_of_two_devices_are_refused(monkeypatch, ops):
    monkeypatch.setattr(ops, "_dev", lambda t: 1 if t.dtype == torch.uint8 else 0)
    with pytest.raises(ops.TfmqError, match="cuda:1"):
        ops.linear_fp8(torch.zeros(4, 40), _pw(ops))


def test_operands_of_the_wrong_form_are_refused(ops):
    from tfmq_dm_amd._lib import TfmqError
    u8, f32 = (lambda *s: torch.zeros(*s, dtype=torch.uint8)), (lambda *s: torch.zeros(*s))      # noqa: E731
    ops.QuantFp8(u8(6, 256), f32(2, 6), (2, 3, 200), torch.float16)
    for q, s in ((u8(5, 256), f32(2, 6)), (u8(6, 128), f32(2, 6)), (u8(6, 256), f32(6, 2)), (u8(6, 256), f32(2, 6).double()), (u8(6, 256).t().contiguous().t(), f32(2, 6))):
        with pytest.raises(TfmqError, match="QuantFp8"):
            ops.QuantFp8(q, s, (2, 3, 200), torch.float16)
    ops.PackedFp8(u8(130, 256), u8(200, 256), f32(2, 2), f32(130), 130, 200)
    for q, qt, s, b in ((u8(130, 200), u8(200, 256), f32(2, 2), None), (u8(130, 256), u8(256, 200), f32(2, 2), None), (u8(130, 256), u8(200, 256), f32(2, 1), None),
                        (u8(130, 256), u8(200, 256), f32(2, 2), f32(129))):
        with pytest.raises(TfmqError, match="PackedFp8"):
            ops.PackedFp8(q, qt, s, b, 130, 200)
