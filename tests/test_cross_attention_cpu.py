"""Refusals of ops.cross_attention / cross_attention_bwd: raised on the host, before anything is launched (no GPU: the handle is a fake)."""
import pytest
import torch

F16 = torch.float16


@pytest.fixture
def ops(monkeypatch):
    import tfmq_dm_amd.ops as ops

    class Never:
        def call(self, name, *a):
            raise AssertionError(f"{name} was launched")
    monkeypatch.setattr(ops, "_dev", lambda t: 0)
    monkeypatch.setattr(ops, "_lib_handle", lambda d=0, p=0: Never())
    return ops


def _z(*s, dt=F16):
    return torch.zeros(*s, dtype=dt)


def test_cpu_tensors_are_refused():
    import tfmq_dm_amd.ops as ops
    with pytest.raises(ops.TfmqError, match="no CPU fallback"):
        ops.cross_attention(_z(1, 2, 64), _z(1, 3, 64), _z(1, 3, 64), 2, 1.0)


BASE = dict(q=(2, 5, 64), k=(2, 7, 64), v=(2, 7, 64), heads=2, scale=1.0)


@pytest.mark.parametrize("change,why", [
    (dict(q=_z(2, 5, 64, dt=torch.float32)), "fp16 or bf16"),
    (dict(k=_z(2, 7, 64, dt=torch.bfloat16)), "k: expected"),
    (dict(k=_z(3, 7, 64)), "k: expected"),
    (dict(v=_z(2, 6, 64)), "v: expected"),
    (dict(q=_z(5, 64)), "must be"),
    (dict(heads=3), "do not split"),
    (dict(heads=4, kv_heads=3), "do not split"),
    (dict(kv_heads=0), "do not split"),
    (dict(kv_heads=1), "k: expected"),
    (dict(q=_z(2, 5, 24), k=_z(2, 7, 24), v=_z(2, 7, 24)), "head dim 12"),
    (dict(q=_z(2, 5, 336), k=_z(2, 7, 336), v=_z(2, 7, 336)), "head dim 168"),
    (dict(q=_z(2, 64, 5).transpose(1, 2)), "unit channel stride"),
    (dict(k=_z(2, 7, 65)[..., 1:]), "aligned"),
    (dict(v=_z(2, 7, 68)[..., :64]), "aligned"),
    (dict(k=torch.empty_strided((2, 2, 64), (1 << 24, 1 << 23, 1), dtype=F16, device="meta"), v=_z(2, 2, 64)), "token strides"),
    (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=float("inf")), "scale"), (dict(scale=float("nan")), "scale"),
    (dict(kv_lens=torch.zeros(2, dtype=torch.int64)), "kv_lens"),
    (dict(kv_lens=torch.zeros(3, dtype=torch.int32)), "kv_lens"),
    (dict(q_lens=torch.zeros(4, dtype=torch.int32)[::2]), "q_lens"),
    (dict(mask=torch.zeros(2, 7)), "mask"),
    (dict(mask=torch.zeros(2, 5, dtype=torch.bool)), "mask"),
    (dict(mask=torch.zeros(7, 2, dtype=torch.bool).t()), "mask"),
])
def test_refusals(ops, change, why):
    a = {n: (_z(*x) if isinstance(x, tuple) else x) for n, x in BASE.items()} | change
    with pytest.raises(ops.TfmqError, match=why):
        ops.cross_attention(**a)
    with pytest.raises(ops.TfmqError, match=why):
        ops.cross_attention_bwd(o=a["q"], lse=torch.zeros(2, 2, 5), g_o=a["q"], **a)


def test_backward_refusals(ops):
    q, k, lse = _z(2, 5, 64), _z(2, 7, 64), torch.zeros(2, 2, 5)
    for o, ls, go, why in ((_z(2, 4, 64), lse, q, "o: expected"), (q, lse, _z(2, 5, 64, dt=torch.bfloat16), "g_o: expected"),
                           (q, lse.double(), q, "lse"), (q, torch.zeros(2, 5, 2), q, "lse"), (q, torch.zeros(2, 5, 2).transpose(1, 2), q, "lse"),
                           (q, lse, _z(2, 5, 65)[..., 1:], "aligned")):
        with pytest.raises(ops.TfmqError, match=why):
            ops.cross_attention_bwd(q, k, k, o, ls, go, 2, 1.0)


def test_operands_of_two_devices_are_refused(monkeypatch, ops):
    monkeypatch.setattr(ops, "_dev", lambda t: 1 if t.dtype == torch.bool else 0)
    with pytest.raises(ops.TfmqError, match="cuda:1"):
        ops.cross_attention(_z(2, 5, 64), _z(2, 7, 64), _z(2, 7, 64), 2, 1.0, mask=torch.ones(2, 7, dtype=torch.bool))


def test_descriptor_layout_matches_the_header(tmp_path):
    """ctypes' layout of tfmq_xattn_desc against the C compiler's."""
    import ctypes as C
    import os
    import shutil
    import subprocess
    import tfmq_dm_amd._lib as L
    cc = shutil.which("gcc")
    if cc is None:
        pytest.skip("no C compiler")
    names = [n for n, _ in L.XattnDesc._fields_]
    inc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    src = tmp_path / "l.c"
    src.write_text('#include <stdio.h>\n#include "tfmq_hip.h"\nint main(void){printf("%zu",sizeof(tfmq_xattn_desc));' +
                   "".join(f'printf(" %zu",offsetof(tfmq_xattn_desc,{n}));' for n in names) + "return 0;}\n")
    subprocess.run([cc, "-I", inc, str(src), "-o", str(tmp_path / "l")], check=True)
    import tfmq_dm_amd.ops as ops
    # the packed form that the calls send: the same places (it ends at the last field)
    last = names[-1]
    assert ops._XATTN.size == getattr(L.XattnDesc, last).offset + getattr(L.XattnDesc, last).size
    raw = ops._XATTN.pack(*range(1, 8), 8.0, *range(9, 9 + len(names) - 8))
    back = L.XattnDesc.from_buffer_copy(raw + bytes(C.sizeof(L.XattnDesc) - len(raw)))
    assert [getattr(back, n) for n in names] == list(range(1, len(names) + 1))
    got = [int(x) for x in subprocess.run([str(tmp_path / "l")], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [C.sizeof(L.XattnDesc)] + [getattr(L.XattnDesc, n).offset for n in names]
