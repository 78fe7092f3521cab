"""Host-side checks of the operators between a block's linear layers (gated norm, rotary positions with several axes, attention within sequences):
argument blocks, refusals, the oracle.  No GPU needed."""

import ctypes
import math
import re
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from nunchaku_amd import _native as nv
from oracle import blocks

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
    mirrors = {"svdq_gated_norm_args": nv.GatedNormArgs, "svdq_rotary_axes_args": nv.RotaryAxesArgs, "svdq_self_attention_args": nv.SelfAttentionArgs}
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


def test_norm_refusals(lib):
    i2 = ctypes.c_int64 * 2
    good = nv.GatedNormArgs(input=16, output=16, M=3, K=64, tokens=1, ld_input=64, ld_output=64, residual_scale=1.0, eps=1e-6)
    entry = lib.svdq_gated_norm
    assert entry(None, None) == -1
    for name in ("input", "output"):
        assert b"null" in _refused(entry, good, lib, **{name: None})
    assert b"residual" in _refused(entry, good, lib, residual_out=16, ld_residual_out=64)
    assert b"dtype" in _refused(entry, good, lib, dtype=2)
    for m in (0, -1, 1 << 31):
        assert b"M (" in _refused(entry, good, lib, M=m)
    for k in (0, 4, 60, 32776):
        assert b"K (" in _refused(entry, good, lib, K=k, ld_input=32784, ld_output=32784)
    assert b"input" in _refused(entry, good, lib, ld_input=56)
    assert b"output" in _refused(entry, good, lib, ld_output=68)
    assert b"residual" in _refused(entry, good, lib, residual=16, ld_residual=8)
    assert b"residual_out" in _refused(entry, good, lib, residual=16, ld_residual=64, residual_out=16, ld_residual_out=32)
    for name in ("input", "output", "weight", "branch_weight", "gate", "scale", "shift"):
        assert b"aligned" in _refused(entry, good, lib, **{name: 24})
    for name in ("gate", "scale", "shift"):
        assert b"strides" in _refused(entry, good, lib, **{name: 16, name + "_stride": i2(68, 0)})
        assert b"strides" in _refused(entry, good, lib, **{name: 16, name + "_stride": i2(0, -64)})
    assert b"tokens" in _refused(entry, good, lib, tokens=0)
    assert b"sequences" in _refused(entry, good, lib, cu_seqlens=16, sequences=0)
    assert b"aligned" in _refused(entry, good, lib, cu_seqlens=18, sequences=1)
    for x in (-1.0, math.nan, math.inf):
        assert b"eps" in _refused(entry, good, lib, eps=x)
    for x in (math.nan, math.inf):
        assert b"residual_scale" in _refused(entry, good, lib, residual_scale=x)


def test_rotary_refusals(lib):
    i3, i4, d4 = ctypes.c_int64 * 3, ctypes.c_int64 * 4, ctypes.c_double * 4
    good = nv.RotaryAxesArgs(q=16, k=16, q_out=16, k_out=16, positions=16, batch=2, tokens=3, heads=4, kv_heads=2, head_dim=64, axes=2, axis_dim=i4(16, 32, 0, 0), theta=d4(1e4, 1e4, 0, 0),
                             q_stride=i3(768, 256, 64), k_stride=i3(384, 128, 64), q_out_stride=i3(768, 256, 64), k_out_stride=i3(384, 128, 64), position_stride=i3(6, 2, 1), eps=1e-6)
    entry = lib.svdq_rotary_axes
    assert entry(None, None) == -1
    for name in ("q", "q_out", "positions"):
        assert b"null" in _refused(entry, good, lib, **{name: None})
    assert b"together" in _refused(entry, good, lib, k=None)
    assert b"together" in _refused(entry, good, lib, k=None, k_out=None, norm_k=16)
    assert b"dtype" in _refused(entry, good, lib, dtype=5)
    assert b"position_type" in _refused(entry, good, lib, position_type=3)
    for changes in (dict(batch=0), dict(tokens=0), dict(batch=1 << 16, tokens=1 << 16)):
        assert b"batch" in _refused(entry, good, lib, **changes)
    for changes in (dict(heads=0), dict(kv_heads=0), dict(heads=65536)):
        assert b"heads" in _refused(entry, good, lib, **changes)
    for d in (0, 60, 264):
        assert b"head_dim" in _refused(entry, good, lib, head_dim=d)
    for n in (0, 5):
        assert b"axes" in _refused(entry, good, lib, axes=n)
    for dims in ((16, 0), (16, 31), (-2, 32), (34, 32), (66, 2)):
        assert b"axis_dim" in _refused(entry, good, lib, axis_dim=i4(*dims, 0, 0)) or b"channels" in lib.svdq_last_error()
    assert b"halves" in _refused(entry, good, lib, axis_dim=i4(16, 24, 0, 0), halves=1)
    for t in (0.0, -1.0, math.nan, math.inf):
        assert b"theta" in _refused(entry, good, lib, theta=d4(1e4, t, 0, 0))
    for name in ("q_stride", "k_stride", "q_out_stride", "k_out_stride"):
        assert b"strides" in _refused(entry, good, lib, **{name: i3(768, 256, 68)})
        assert b"strides" in _refused(entry, good, lib, **{name: i3(-768, 256, 64)})
    assert b"positions" in _refused(entry, good, lib, position_stride=i3(-6, 2, 1))
    for name in ("q", "k", "q_out", "k_out", "norm_q", "norm_k"):
        assert b"aligned" in _refused(entry, good, lib, **{name: 24})
    assert b"aligned" in _refused(entry, good, lib, positions=18)
    assert b"aligned" in _refused(entry, good, lib, positions=20, position_type=1)
    assert b"eps" in _refused(entry, good, lib, eps=math.nan)


def test_attention_refusals(lib):
    i3 = ctypes.c_int64 * 3
    good = nv.SelfAttentionArgs(q=16, k=16, v=16, out=16, batch=2, heads=4, kv_heads=2, head_dim=64, q_len=3, k_len=5, q_stride=i3(768, 256, 64),
                                k_stride=i3(640, 128, 64), v_stride=i3(640, 128, 64), out_stride=i3(768, 256, 64), scale=0.125)
    need = ctypes.c_int64()
    for entry in (lib.svdq_self_attention, lambda a, _: lib.svdq_self_attention_workspace(a, ctypes.byref(need))):
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
        assert b"at most one" in _refused(entry, good, lib, key_lengths=16, cu_seqlens_k=16)
        for s in (0.0, -1.0, math.inf, math.nan):
            assert b"scale" in _refused(entry, good, lib, scale=s)
        for name in ("q_stride", "k_stride", "v_stride", "out_stride"):
            assert b"strides" in _refused(entry, good, lib, **{name: i3(768, 256, 68)})
            assert b"strides" in _refused(entry, good, lib, **{name: i3(-768, 256, 64)})
        assert b"apart" in _refused(entry, good, lib, k_stride=i3(0, 1 << 24, 64))
        assert b"aligned" in _refused(entry, good, lib, v=24)
        for name in ("key_lengths", "cu_seqlens_q", "cu_seqlens_k"):
            assert b"aligned" in _refused(entry, good, lib, **{name: 18})


def test_wrappers_refuse_cpu_tensors():
    from nunchaku_amd import ops

    x, q, p = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(1, 4, 2, 64, dtype=torch.bfloat16), torch.zeros(4, 1, dtype=torch.int32)
    for call in (lambda: ops.gated_norm(x), lambda: ops.rotary_axes(q, q, p, (64,)), lambda: ops.self_attention(q, q, q)):
        with pytest.raises(RuntimeError, match="GPU"):
            call()


def test_oracle_by_hand():
    """Literals: a quarter turn, a norm of (3, 4), three causal rows with softmax weights of 1 : 3."""
    x = torch.tensor([[3.0, 4.0]], dtype=torch.bfloat16)
    y, h, _ = blocks.gated_norm(x, x, "rms", gate=torch.tensor([1.0, 0.0]), shift=torch.tensor([0.0, 1.0]), residual_scale=2.0, eps=0.0)
    assert h.tolist() == [[9.0, 8.0]] and torch.allclose(y, torch.tensor([[9.0, 8.0]], dtype=torch.float64) / math.sqrt(72.5) + torch.tensor([0.0, 1.0]))
    y, _, _ = blocks.gated_norm(x, None, "layer", scale=torch.tensor([1.0, 0.0]), eps=0.0)
    assert torch.allclose(y, torch.tensor([[-2.0, 1.0]], dtype=torch.float64))
    # theta 16 over four channels: frequencies 1 and 1 / 4
    q = torch.tensor([1.0, 0.0, 1.0, 0.0], dtype=torch.float64).view(1, 1, 4)
    y, size = blocks.rotary(q, torch.tensor([[2 * math.pi]], dtype=torch.float64), (4,), theta=16.0)
    assert torch.allclose(y.flatten(), torch.tensor([1.0, 0.0, 0.0, 1.0], dtype=torch.float64), atol=1e-12) and size.flatten().tolist() == [1.0] * 4
    y, _ = blocks.rotary(q, torch.tensor([[math.pi / 2]], dtype=torch.float64), (4,), theta=16.0, interleaved=False)  # pairs (0, 2), (1, 3)
    assert torch.allclose(y.flatten(), torch.tensor([-1.0, 0.0, 1.0, 0.0], dtype=torch.float64), atol=1e-12)
    assert blocks.angles(torch.tensor([[3.0, 5.0]]), (2, 2), 16.0, "head").tolist() == [[3.0, 1.25]]
    q = torch.ones(2, 1, 1, dtype=torch.float64)
    k = torch.tensor([0.0, math.log(3.0), 7.0], dtype=torch.float64).view(3, 1, 1)
    v = torch.tensor([4.0, 8.0, math.nan], dtype=torch.float64).view(3, 1, 1)
    out = blocks.self_attention(q, k, v, True, 1.0)
    assert abs(out[0].item() - 7.0) < 1e-12 and out[1].isnan().all()
    assert blocks.self_attention(q, k[:1], v[:1], True, 1.0).flatten().tolist() == [0.0, 4.0]
