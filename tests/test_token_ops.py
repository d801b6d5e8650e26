"""CPU: the token operators' host side -- descriptor layouts, refusals, frequency tables -- and their oracle (the generator's published vectors, the
backward formulas against differences).  No kernel runs here."""
import ctypes as C
import math
import os
import subprocess

import numpy as np
import pytest
import torch

from oracle import token_oracle as O
from yolopoint_amd import _hip
from yolopoint_amd.utils import token_ops as ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_descriptors_match_the_header(tmp_path):
    """The ctypes layouts against what the C compiler makes of include/yolopoint_hip.h."""
    fields = [("YpLayerNormDesc", f[0]) for f in _hip.YpLayerNormDesc._fields_] + [("YpRotaryDesc", f[0]) for f in _hip.YpRotaryDesc._fields_]
    src = tmp_path / "size.c"
    src.write_text('#include "yolopoint_hip.h"\n#include <stdio.h>\nint main(void) { printf("%zu %zu", sizeof(YpLayerNormDesc), sizeof(YpRotaryDesc));\n'
                   + "".join(f'printf(" %zu", offsetof({s}, {f}));\n' for s, f in fields) + "return 0; }\n")
    exe = tmp_path / "size"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [C.sizeof(_hip.YpLayerNormDesc), C.sizeof(_hip.YpRotaryDesc)] + [getattr(getattr(_hip, s), f).offset for s, f in fields]


def norm_desc(rows, D, dtype, wdtype=_hip.YP_F32, p=0.0, **more):
    return C.byref(_hip.YpLayerNormDesc(rows=rows, D=D, dtype=dtype, wdtype=wdtype, eps=0.1, p=p, **more))


def test_entry_points_refuse_bad_descriptors():
    """Checked on the host before anything is launched (no GPU here)."""
    l = _hip.lib()
    n, f16, f32, widest = norm_desc, _hip.YP_F16, _hip.YP_F32, 16384
    assert l.yp_layer_norm_fwd(None, None) == -1 and l.yp_layer_norm_bwd(None, None) == -1 and l.yp_rotary(None, None) == -1
    for bad in (n(-1, 8, f16, f32, x=64, y=64), n(4, 0, f16, f32, x=64, y=64), n(4, widest + 1, f16, f32, x=64, y=64),
                n(4, 8, f32, f16, x=64, y=64), n(4, 8, f16, f32, y=64), n(4, 8, f16, f32, x=64), n(4, 8, f16, f32, x=64, y=64, res=64),
                n(4, 8, f16, f32, x=64, y=64, mean=64), n(4, 8, f16, f32, 0.5, x=64, y=64), n(4, 8, f16, f32, 1.5, x=64, y=64, res=64, z=64),
                n(4, 8, f16, f32, float("nan"), x=64, y=64, res=64, z=64), n(4, 8, f16, f32, x=64, y=64, x_stride=-1)):
        assert l.yp_layer_norm_fwd(bad, None) == -1
    ok = dict(x=64, dy=64, mean=64, rstd=64, dres=64)
    for bad in (n(4, 8, f16, f32, **{**ok, "dy": 0}), n(4, 8, f16, f32, **{**ok, "mean": 0}), n(4, 8, f16, f32, 0.5, **ok), n(4, 8, f16, f32, dz_stride=-8, **ok)):
        assert l.yp_layer_norm_bwd(bad, None) == -1
    assert l.yp_layer_norm_bwd(n(4, 8, f16, f32, dweight=64, **ok), None) == -4                       # no workspace
    assert l.yp_layer_norm_bwd(n(4, 8, f16, f32, dweight=64, workspace=64, workspace_bytes=16, **ok), None) == -4
    assert l.yp_layer_norm_bwd_workspace_bytes(4, 8, _hip.YP_F16) >= 2 * 8 * 4
    assert [l.yp_layer_norm_bwd_workspace_bytes(*a) for a in ((0, 8, 0), (4, 0, 0), (4, 8, 9))] == [0, 0, 0]
    assert l.yp_layer_norm_fwd(n(0, 8, f16, f32), None) == 0                                          # nothing to do
    assert l.yp_layer_norm_max_width(_hip.YP_F32) == widest and l.yp_layer_norm_max_width(7) == 0
    for bad in ((64, None, 64, 8, 7, 0.1), (64, None, 64, 8, 0, -0.1), (64, None, 64, 8, 0, 1.1), (64, None, 64, -1, 0, 0.1), (None, None, 64, 8, 0, 0.1), (64, None, None, 8, 0, 0.1)):
        assert l.yp_dropout(*bad, 0, 0, None, None) == -1
    assert l.yp_dropout(None, None, None, 0, 0, 0.1, 0, 0, None, None) == 0

    def rot(q=64, k=0, qo=64, ko=0, pos=64, f=64, B=1, T=4, Hq=2, Hk=0, D=8, R=8, dt=0, pt=0, axes=1):
        return C.byref(_hip.YpRotaryDesc(q=q, k=k, q_out=qo, k_out=ko, positions=pos, inv_freq=f, B=B, T=T, Hq=Hq, Hk=Hk, D=D, R=R, dtype=dt, position_type=pt, axes=axes, scale=1.0))
    for bad in (rot(dt=7), rot(B=-1), rot(B=1 << 16, T=1 << 15), rot(D=1, R=1), rot(D=1026), rot(R=7), rot(R=10), rot(R=0), rot(axes=3), rot(R=6, axes=2), rot(pt=5), rot(q=0),
                rot(Hk=1), rot(f=0), rot(pos=0, axes=2)):
        assert l.yp_rotary(bad, None) == -1
    assert l.yp_rotary(rot(q=0, T=0), None) == 0 and l.yp_last_error()


def test_cpu_tensors_are_refused():
    x = torch.randn(4, 8)
    with pytest.raises(_hip.YpError):
        ops.layer_norm(x)
    with pytest.raises(_hip.YpError):
        ops.dropout(x, 0.1, (0, 0))
    with pytest.raises(_hip.YpError):
        ops.dropout_add_layer_norm(x, x)
    with pytest.raises(_hip.YpError):
        ops.rotary(x.view(1, 1, 4, 8), 0, torch.ones(4, dtype=torch.float64))
    with pytest.raises(_hip.YpError):
        ops.layer_norm("x")


def test_philox_known_answers():
    """The published vectors of Philox4x32-10 (Random123's kat_vectors)."""
    def run(ctr, key):
        lo, hi = ctr[0] | ctr[1] << 32, ctr[2] | ctr[3] << 32
        return [int(v) for v in O.philox4x32_10((np.array([lo], np.uint64), np.array([hi], np.uint64)), key[0] | key[1] << 32)[0]]
    f = 0xFFFFFFFF
    assert run((0, 0, 0, 0), (0, 0)) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert run((f, f, f, f), (f, f)) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    assert run((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0)) == [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]


def test_oracle_mask_is_indexed_by_the_flat_element():
    whole = O.keep_mask(1000, 0.3, 5, 9)
    assert torch.equal(whole[137:300], O.keep_mask(163, 0.3, 5, 9, start=137))
    assert not torch.equal(whole, O.keep_mask(1000, 0.3, 5, 10)) and not torch.equal(whole, O.keep_mask(1000, 0.3, 6, 9))
    big = O.keep_mask(1 << 20, 0.3, 1, 2).double().mean()
    assert abs(float(big) - 0.7) < 5 * math.sqrt(0.21 / (1 << 20))                     # five standard deviations


def test_oracle_gradients_against_differences():
    """layer_norm_backward and rotary's turning back against central differences of the forward definitions (64 bits: h^2 and 1e-16 / h)."""
    g = torch.Generator().manual_seed(3)
    x, w, b = torch.randn(3, 7, generator=g).double(), torch.randn(7, generator=g).double(), torch.randn(7, generator=g).double()
    dy = torch.randn(3, 7, generator=g).double()
    h = 1e-5

    def slope(f, t):
        out = torch.empty_like(t)
        for i in range(t.numel()):
            up, down = t.clone(), t.clone()
            up.view(-1)[i] += h
            down.view(-1)[i] -= h
            out.view(-1)[i] = (f(up) - f(down)) / (2 * h)
        return out
    dx, dw, db = O.layer_norm_backward(x, w, dy, 1e-5)
    assert torch.allclose(dx, slope(lambda t: (O.layer_norm(t, w, b, 1e-5)[0] * dy).sum(), x), rtol=1e-6, atol=1e-8)
    assert torch.allclose(dw, slope(lambda t: (O.layer_norm(x, t, b, 1e-5)[0] * dy).sum(), w), rtol=1e-6, atol=1e-8)
    assert torch.allclose(db, slope(lambda t: (O.layer_norm(x, w, t, 1e-5)[0] * dy).sum(), b), rtol=1e-6, atol=1e-8)
    q, pos, f = torch.randn(1, 2, 1, 6, generator=g).double(), torch.tensor([3.0, 11.0]), torch.tensor([1.0, 0.1]).double()
    dq = torch.randn(1, 2, 1, 6, generator=g).double()
    for inter in (False, True):
        back = O.rotary(dq, pos, f, inter, "bthd", 1.25, inverse=True)
        assert torch.allclose(back, slope(lambda t: (O.rotary(t, pos, f, inter, "bthd", 1.25) * dq).sum(), q), rtol=1e-6, atol=1e-8)


def test_frequency_tables():
    f, s = ops.rotary_frequencies(8, 10000.0)
    assert f.dtype == torch.float64 and s == 1.0 and torch.allclose(f, 10000.0 ** (-torch.arange(4).double() / 4), rtol=1e-15)
    f2, _ = ops.rotary_frequencies(16, 100.0, axes=2)
    assert torch.equal(f2[:4], f2[4:]) and torch.equal(f2[:4], ops.rotary_frequencies(8, 100.0)[0])
    lin, _ = ops.rotary_frequencies(8, scaling="linear", factor=4.0)
    assert torch.allclose(lin, f / 4, rtol=1e-15)
    ntk, _ = ops.rotary_frequencies(8, scaling="ntk", factor=4.0)
    assert ntk[0] == 1.0 and torch.allclose(ntk[-1], f[-1] / 4, rtol=1e-12)
    yarn, s = ops.rotary_frequencies(128, scaling="yarn", factor=8.0, original=4096)
    f = ops.rotary_frequencies(128)[0]
    turns = 4096 * f / (2 * math.pi)
    assert torch.allclose(yarn[turns > 33], f[turns > 33], rtol=1e-15) and torch.allclose(yarn[turns < 0.9], f[turns < 0.9] / 8, rtol=1e-15)
    assert bool((yarn <= f).all()) and bool((yarn >= f / 8 * (1 - 1e-15)).all()) and s == 0.1 * math.log(8.0) + 1.0
    assert ops.rotary_frequencies(64, scaling="yarn", factor=1.0, original=4096)[1] == 1.0
    for bad in (dict(dim=7), dict(dim=6, axes=2), dict(dim=8, axes=3), dict(dim=0), dict(dim=8, scaling="cubic", factor=2.0), dict(dim=8, factor=2.0),
                dict(dim=8, scaling="linear", factor=0.5), dict(dim=8, scaling="yarn", factor=2.0), dict(dim=8, scaling="yarn", factor=2.0, original=64, fast=1.0, slow=2.0),
                dict(dim=2, scaling="ntk", factor=2.0)):
        with pytest.raises(_hip.YpError):
            ops.rotary_frequencies(**bad)


@pytest.mark.parametrize("dim,axes,base,original,factor", [(128, 1, 10000.0, 262144, 8.0), (128, 1, 10000.0, 4096, 8.0), (64, 2, 100.0, 640, 4.0), (64, 1, 500000.0, 8192, 32.0),
                                                           (64, 2, 100.0, 1 << 20, 4.0), (64, 1, 10000.0, 4, 2.0), (64, 1, 10000.0, 6, 2.0), (2, 1, 10000.0, 640, 2.0)])
def test_yarn_table_against_the_published_formula(dim, axes, base, original, factor):
    """The ramp runs from floor(pair with `fast` turns) >= 0 to ceil(pair with `slow` turns) <= d - 1, wherever the last pair stands; pairs of more than `fast`
    turns stay and pairs of fewer than `slow` are divided by the factor at every length."""
    d, fast, slow = dim // axes, 32.0, 1.0
    f = float(base) ** (-np.arange(d // 2) / (d / 2))
    place = [d * math.log(original / (n * 2 * math.pi)) / (2 * math.log(base)) for n in (fast, slow)]
    low, high = max(math.floor(place[0]), 0), min(math.ceil(place[1]), d - 1)
    turns = original * f / (2 * math.pi)
    want = np.empty(d // 2)
    for j in range(d // 2):
        r = 1.0 if turns[j] < slow else 0.0 if turns[j] > fast else (j - low) / (high - low)
        want[j] = f[j] * (1 - r) + f[j] / factor * r
    got, scale = ops.rotary_frequencies(dim, base, axes=axes, scaling="yarn", factor=factor, original=original)
    # (64 bits: a handful of roundings of 2^-53 each)
    assert got.shape == (dim // 2,) and np.allclose(got.numpy(), np.tile(want, axes), rtol=64 * 2.0 ** -53, atol=0.0) and scale == 0.1 * math.log(factor) + 1.0


def test_frequency_tables_refuse_what_has_no_table():
    inf, nan = math.inf, math.nan
    yarn = dict(dim=8, scaling="yarn", factor=2.0)
    for bad in (dict(dim=8, base=0.0), dict(dim=8, base=-2.0), dict(dim=8, base=nan), dict(dim=8, base=inf), dict(dim=8, base="b"), dict(dim=8.0), dict(dim="8"), dict(dim=8, axes=1.0),
                dict(dim=8, factor=nan), dict(dim=8, scaling="linear", factor=inf), dict(dim=8, scaling="ntk", factor=inf), dict(dim=16, base=1e300, scaling="ntk", factor=1e300),
                dict(yarn, original=-5), dict(yarn, original=inf), dict(yarn, original=nan), dict(yarn, original="x"), dict(yarn, original=64, base=1.0), dict(yarn, original=64, base=0.5),
                dict(yarn, original=64, fast=inf), dict(yarn, original=64, slow=nan), dict(yarn, original=64, factor="y"), dict(dim=8, base=10 ** 400)):
        with pytest.raises(_hip.YpError):
            ops.rotary_frequencies(**bad)
    # what was a table stays one
    assert torch.equal(ops.rotary_frequencies(np.int64(8), 1.0)[0], torch.ones(4, dtype=torch.float64)) and ops.rotary_frequencies(8, 0.25)[0][1] == 0.25 ** -0.25


def traced_calls(inv):
    return {"layer_norm": lambda t: ops.layer_norm(t), "dropout_add_layer_norm": lambda t: ops.dropout_add_layer_norm(t, t)[0], "dropout": lambda t: ops.dropout(t, 0.5, (1, 2)),
            "rotary": lambda t: ops.rotary(t.view(1, 1, *t.shape), 0, inv)}


@pytest.mark.parametrize("op", ["layer_norm", "dropout_add_layer_norm", "dropout", "rotary"])
def test_traced_calls_are_refused(op):
    """A recording would hold the empty buffers of the results and not what fills them."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    x, inv = torch.randn(4, 8), ops.rotary_frequencies(8)[0]
    f = traced_calls(inv)[op]
    with pytest.raises(_hip.YpError, match="cannot be traced"):
        torch.jit.trace(f, x)
    with pytest.raises(_hip.YpError, match="cannot be traced"):
        make_fx(f)(x)
    with pytest.raises(_hip.YpError, match="cannot be traced"), FakeTensorMode(allow_non_fake_inputs=True):
        f(x)
    with pytest.raises(_hip.YpError, match="on the GPU"):
        f(x)


class Wrapper(torch.Tensor):
    """A tensor that says where it lies and holds nothing there, as sharded parameters do."""
    @staticmethod
    def __new__(cls, shape, dtype, device):
        return torch.Tensor._make_wrapper_subclass(cls, shape, dtype=dtype, device=device)

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise RuntimeError(f"{func} was called on a wrapper")


def test_tensors_without_memory_are_refused():
    x, inv = Wrapper((4, 8), torch.float32, "cuda:0"), ops.rotary_frequencies(8)[0]
    for call in (lambda: ops.layer_norm(x), lambda: ops.dropout(x, 0.5, (1, 2)), lambda: ops.dropout_add_layer_norm(x, x),
                 lambda: ops.rotary(Wrapper((1, 2, 3, 8), torch.float32, "cuda:0"), 0, inv)):
        with pytest.raises(_hip.YpError, match="memory"):
            call()


def test_rotary_refuses_head_counts_past_32_bits():
    """A thread steps over the heads in 32 bits: a sum of heads near 2^31 would wrap to heads before the first."""
    l = _hip.lib()
    for Hq, Hk, B, T in (((1 << 30) + 1, 0, 1, 1), (1 << 30, 1, 1, 1), ((1 << 30) - 1, (1 << 30) - 1, 1, 1), ((1 << 31) - 1, (1 << 31) - 1, 1, 1), ((1 << 31) - 1, 1, 1, 4),
                         (1 << 30, 0, 1 << 10, 1 << 20)):
        d = _hip.YpRotaryDesc(q=64, k=64, q_out=64, k_out=64, positions=64, inv_freq=64, B=B, T=T, Hq=Hq, Hk=Hk, D=2, R=2, axes=1, scale=1.0)
        assert l.yp_rotary(C.byref(d), None) == -1 and b"heads" in l.yp_last_error()


def test_the_library_builds_without_torch():
    """`make` for a C program: no torch, no Python headers."""
    def commands(*more):
        return subprocess.run(["make", "-n", "-B", "-C", os.path.join(ROOT, "yolopoint_amd", "csrc"), *more, "all"], check=True, capture_output=True, text=True)
    bare, full = commands("PYTHON=/bin/false"), commands()
    assert "libyolopoint_hip.so" in bare.stdout and "token_autograd" not in bare.stdout and "Traceback" not in bare.stderr
    assert "libyolopoint_hip.so" in full.stdout and "token_autograd.cpp" in full.stdout


def test_build_compiles_where_a_library_is_there(monkeypatch):
    import __graft_entry__ as entry
    calls = []
    monkeypatch.setattr(entry.subprocess, "run", lambda cmd, **kw: calls.append(cmd))
    entry.build()
    assert calls[0][0] == "make" and "-B" in calls[0]


def test_no_build_of_the_kernels_has_packed_fp32():
    """Every compiled object, of the library and of the sanitizer's, leaves those instructions out."""
    for goal in ("all", "asan"):
        out = subprocess.run(["make", "-n", "-B", "-C", os.path.join(ROOT, "yolopoint_amd", "csrc"), goal], check=True, capture_output=True, text=True).stdout
        lines = [l for l in out.splitlines() if ".hip -o" in l]
        assert len(lines) >= 14 and all("-Xclang -target-feature -Xclang -packed-fp32-ops" in l for l in lines), goal


def test_the_version_rose_with_the_descriptor(tmp_path):
    """A program built against an earlier header passes a shorter YpLayerNormDesc: it can tell by the version."""
    src = tmp_path / "version.c"
    src.write_text('#include "yolopoint_hip.h"\n#include <stdio.h>\nint main(void) { printf("%d %zu %zu", YP_VERSION, offsetof(YpLayerNormDesc, stats), sizeof(YpLayerNormDesc)); return 0; }\n')
    exe = tmp_path / "version"
    subprocess.run(["gcc", "-include", "stddef.h", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    version, offset, size = (int(v) for v in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split())
    assert _hip.lib().yp_version() == version >= 101 and offset + C.sizeof(C.c_void_p) == size
