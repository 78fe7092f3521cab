"""Host-side checks of the 8-bit linear operators and of attention to an encoder's states: argument blocks, refusals, the layer
module, the oracle.  No GPU needed."""

import ctypes
import math
import re
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from nunchaku_amd import _native as nv
from oracle import w8a8 as ow

ROOT = Path(__file__).resolve().parents[1]


@pytest.fixture(scope="module")
def lib():
    if not nv.LIB_PATH.exists():
        nv.build()
    return nv.lib()


def test_mirrors_match_the_header(tmp_path):
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no host C compiler")
    header = ROOT / "include" / "svdq_amd.h"
    mirrors = {"svdq_quantize_w8a8_args": nv.QuantizeW8A8Args, "svdq_gemm_w8a8_args": nv.GemmW8A8Args, "svdq_cross_attention_args": nv.CrossAttentionArgs}
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{header}"', "int main(void) {"]
    for cname, mirror in mirrors.items():
        lines.append(f'printf("{cname} %zu\\n", sizeof({cname}));')
        lines += [f'printf("{cname}.{f} %zu\\n", offsetof({cname}, {f}));' for f, *_ in mirror._fields_]
    (tmp_path / "layout.c").write_text("\n".join([*lines, "return 0; }"]))
    subprocess.run([cc, str(tmp_path / "layout.c"), "-o", str(tmp_path / "layout")], check=True, capture_output=True)
    out = dict(line.split() for line in subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.splitlines())
    text = header.read_text()
    for cname, mirror in mirrors.items():
        assert int(out[cname]) == ctypes.sizeof(mirror), cname
        for f, *_ in mirror._fields_:
            assert int(out[f"{cname}.{f}"]) == getattr(mirror, f).offset, f"{cname}.{f}"
        body = re.sub(r"/\*.*?\*/", "", text[text.index(f"typedef struct {cname}"):text.index(f"}} {cname};")], flags=re.S)
        assert set(re.findall(r"[\s\*]([A-Za-z_][A-Za-z0-9_]*)\s*(?:\[\d+\])?\s*[,;]", body)) == {f[0] for f in mirror._fields_}, cname


def _refused(entry, good, lib, **changes):
    bad = type(good).from_buffer_copy(good)
    for k, v in changes.items():
        setattr(bad, k, v)
    assert entry(ctypes.byref(bad), None) == -1, changes
    return lib.svdq_last_error()


def test_quantize_refusals(lib):
    good = nv.QuantizeW8A8Args(input=16, weight=16, output=16, oscales=16, M=3, K=64, ld_input=64, eps=1e-6)
    for entry in (lib.svdq_quantize_w8a8_act, lib.svdq_rms_norm_quantize_w8a8):
        assert entry(None, None) == -1
        for name in ("input", "output", "oscales"):
            assert b"null" in _refused(entry, good, lib, **{name: None})
        assert b"K" in _refused(entry, good, lib, K=24)
        assert b"K" in _refused(entry, good, lib, K=65552, ld_input=65552)
        assert b"K" in _refused(entry, good, lib, K=0)
        assert b"M" in _refused(entry, good, lib, M=0)
        assert b"M" in _refused(entry, good, lib, M=1 << 31)
        assert b"input" in _refused(entry, good, lib, ld_input=56)
        assert b"input" in _refused(entry, good, lib, ld_input=68)
        assert b"aligned" in _refused(entry, good, lib, input=8)
        assert b"aligned" in _refused(entry, good, lib, oscales=18)
        assert b"dtype" in _refused(entry, good, lib, dtype=2)
        assert b"residual" in _refused(entry, good, lib, residual=16)
    norm = lib.svdq_rms_norm_quantize_w8a8
    assert b"weight" in _refused(norm, good, lib, weight=None)
    assert b"eps" in _refused(norm, good, lib, eps=-1.0)
    assert b"eps" in _refused(norm, good, lib, eps=math.nan)
    assert b"residual" in _refused(norm, good, lib, residual=16, residual_out=16, ld_residual=32, ld_residual_out=64)
    assert b"residual_out" in _refused(norm, good, lib, residual=16, residual_out=16, ld_residual=64, ld_residual_out=32)
    assert b"residual" in _refused(lib.svdq_quantize_w8a8_act, good, lib, residual=16, residual_out=16, ld_residual=64, ld_residual_out=64)


def test_gemm_refusals(lib):
    good = nv.GemmW8A8Args(act=16, wgt=16, ascales=16, wscales=16, out=16, M=3, N=5, K=64, ld_act=64, ld_wgt=64, ld_out=5)
    need = ctypes.c_int64()
    for entry in (lib.svdq_gemm_w8a8, lambda a, _: lib.svdq_gemm_w8a8_workspace(a, ctypes.byref(need))):
        _gemm_refusals(entry, good, lib)


def _gemm_refusals(entry, good, lib):
    assert entry(None, None) == -1
    for name in ("act", "wgt", "ascales", "wscales", "out"):
        assert b"null" in _refused(entry, good, lib, **{name: None})
    for changes in (dict(M=0), dict(N=0), dict(M=1 << 31), dict(N=1 << 31)):
        assert b"M (" in _refused(entry, good, lib, **changes)
    for changes in (dict(M=(1 << 29) + 1, N=1), dict(M=33, N=1 << 28), dict(M=1 << 20, N=1 << 15, ld_out=1 << 15)):
        assert b"M (" in _refused(entry, good, lib, **changes) or b"outputs" in _refused(entry, good, lib, **changes)
    for k in (0, 8, 72, 131072):
        assert b"K (" in _refused(entry, good, lib, K=k, ld_act=131072, ld_wgt=131072)
    assert b"act" in _refused(entry, good, lib, ld_act=48)
    assert b"act" in _refused(entry, good, lib, ld_act=72)
    assert b"act" in _refused(entry, good, lib, ld_act=1 << 23)
    assert b"wgt" in _refused(entry, good, lib, ld_wgt=1 << 23)
    assert b"out" in _refused(entry, good, lib, ld_out=4)
    assert b"aligned" in _refused(entry, good, lib, act=8)
    assert b"aligned" in _refused(entry, good, lib, wscales=18)
    assert b"dtype" in _refused(entry, good, lib, dtype=-1)


def test_attention_refusals(lib):
    i3 = ctypes.c_int64 * 3
    good = nv.CrossAttentionArgs(q=16, k=16, v=16, out=16, batch=2, heads=4, kv_heads=2, head_dim=64, q_len=3, k_len=5, q_stride=i3(768, 256, 64),
                                 k_stride=i3(640, 128, 64), v_stride=i3(640, 128, 64), out_stride=i3(768, 256, 64), scale=0.125)
    need = ctypes.c_int64()
    for entry in (lib.svdq_cross_attention, lambda a, _: lib.svdq_cross_attention_workspace(a, ctypes.byref(need))):
        assert entry(None, None) == -1
        for name in ("q", "k", "v", "out"):
            assert b"null" in _refused(entry, good, lib, **{name: None})
        assert b"dtype" in _refused(entry, good, lib, dtype=7)
        for changes in (dict(batch=0), dict(heads=0), dict(kv_heads=0), dict(kv_heads=3), dict(batch=65536)):
            assert b"batch" in _refused(entry, good, lib, **changes)
        for d in (0, 4, 60, 136):
            assert b"head_dim" in _refused(entry, good, lib, head_dim=d)
        assert b"q_len" in _refused(entry, good, lib, q_len=0)
        assert b"k_len" in _refused(entry, good, lib, k_len=0)
        assert b"k_len" in _refused(entry, good, lib, k_len=1 << 31)
        assert b"q_len" in _refused(entry, good, lib, q_len=1 << 30)
        assert b"too many" in _refused(entry, good, lib, batch=65535, heads=512, kv_heads=512)
        assert b"too many" in _refused(entry, good, lib, q_len=1 << 28)
        assert b"at most one" in _refused(entry, good, lib, key_lengths=16, key_mask=16)
        assert b"at most one" in _refused(entry, good, lib, key_lengths=16, cu_seqlens_k=16)
        for s in (0.0, -1.0, math.inf, math.nan):
            assert b"scale" in _refused(entry, good, lib, scale=s)
        for name in ("q_stride", "k_stride", "v_stride", "out_stride"):
            assert b"strides" in _refused(entry, good, lib, **{name: i3(768, 256, 68)})
            assert b"strides" in _refused(entry, good, lib, **{name: i3(-768, 256, 64)})
        assert b"apart" in _refused(entry, good, lib, k_stride=i3(0, 1 << 24, 64))
        assert b"aligned" in _refused(entry, good, lib, v=24)
        assert b"aligned" in _refused(entry, good, lib, key_lengths=18)


def test_wrappers_refuse_cpu_tensors():
    from nunchaku_amd import ops

    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    q = torch.zeros(1, 4, 2, 64, dtype=torch.bfloat16)
    c = torch.zeros(4, 64, dtype=torch.int8)
    for call in (lambda: ops.quantize_w8a8_act(x), lambda: ops.rms_norm_quantize_w8a8(x, x[0]), lambda: ops.gemm_w8a8(c, c, x, x), lambda: ops.cross_attention(q, q, q)):
        with pytest.raises(RuntimeError, match="GPU"):
            call()


def test_layer_quantizes_its_weights():
    from nunchaku_amd.models import W8A8Linear

    torch.manual_seed(0)
    lin = torch.nn.Linear(96, 40, dtype=torch.bfloat16)
    with torch.no_grad():
        lin.weight[3] = 0
    m = W8A8Linear.from_linear(lin)
    codes, scales = ow.quantize_rows(lin.weight.detach())
    assert torch.equal(m.qweight, codes) and torch.equal(m.wscales, scales) and torch.equal(m.bias, lin.bias)
    assert m.bias.dtype == torch.bfloat16 and not any(p.requires_grad for p in m.parameters())
    # every weight within half a step of what its code stands for (1.001: the steps' own roundings)
    assert ((m.qweight.float() * m.wscales[:, None] - lin.weight.float()).abs() <= 0.5005 * m.wscales[:, None]).all()
    again = W8A8Linear(96, 40)
    again.load_state_dict(m.state_dict())
    assert torch.equal(again.qweight, codes)
    assert "bias" not in W8A8Linear(96, 40, bias=False).state_dict()
    with pytest.raises(ValueError, match="multiple of 16"):
        W8A8Linear(100, 40)
    with torch.no_grad():
        lin.weight[0, 0] = math.inf
    with pytest.raises(ValueError, match="infinities"):
        W8A8Linear.from_linear(lin)


def test_layer_keeps_its_scales_when_the_model_is_cast():
    from nunchaku_amd.models import W8A8Linear

    torch.manual_seed(1)
    m = W8A8Linear.from_linear(torch.nn.Linear(96, 40))  # fp32: the operators' default type
    assert m.torch_dtype == m.bias.dtype == torch.bfloat16
    scales, codes = m.wscales.clone(), m.qweight.clone()
    model = torch.nn.Sequential(m, torch.nn.Linear(40, 8)).to(torch.float16)
    assert model[1].weight.dtype == m.bias.dtype == m.torch_dtype == torch.float16
    assert torch.equal(m.wscales, scales) and m.wscales.dtype == torch.float32 and isinstance(m.wscales, torch.nn.Parameter)
    assert torch.equal(model.double()[0].wscales, scales) and torch.equal(m.qweight, codes)
    assert m.to("meta").wscales.dtype == torch.float32


def test_oracle_by_hand():
    """Literals: a tie goes to the even code, the floor keeps a row of zeros, a bad row is NaN, and softmax weights of 1 : 3."""
    codes, scales = ow.quantize_rows(torch.tensor([[127.0, 0.5, 1.5, -2.5], [0.0, 0.0, 0.0, 0.0], [1.0, math.inf, 2.0, 3.0], [math.nan, 1.0, 1.0, 1.0]]))
    assert codes.tolist() == [[127, 0, 2, -2], [0] * 4, [0] * 4, [0] * 4]
    assert scales[0] == 1.0 and 0 < scales[1] < 1e-30 and torch.isnan(scales[2:]).all()
    q = torch.ones(1, 1, 1, 1, dtype=torch.float64)
    k = torch.tensor([0.0, math.log(3.0), 9.0], dtype=torch.float64).view(1, 3, 1, 1)
    v = torch.tensor([4.0, 8.0, math.nan], dtype=torch.float64).view(1, 3, 1, 1)
    assert abs(ow.cross_attention(q, k, v, torch.tensor([[True, True, False]]), 1.0).item() - 7.0) < 1e-12
    assert ow.cross_attention(q, k, v, torch.zeros(1, 3, dtype=torch.bool)).item() == 0.0
    x, w = torch.tensor([[3.0, 4.0]], dtype=torch.bfloat16), torch.tensor([2.0, 1.0], dtype=torch.bfloat16)
    codes, scales, h = ow.rms_norm_quantize(x, w, eps=0.0)
    assert codes.tolist() == [[127, 85]] and abs(scales.item() - 6.0 / math.sqrt(12.5) / 127.0) < 1e-15 and torch.equal(h, x)
