#!/usr/bin/env python3
"""Measurements of the token operators (yolopoint_amd/utils/token_ops.py) on one MI355X; what profiles/token_ops_rates.txt and token_ops_kernels.txt hold.

  python tools/token_bench.py rates                 each operator over widths, types and layouts (tensors of 128 MiB): time and TB/s
  python tools/token_bench.py copies                a torch copy by size and a large bf16 product: what the card reaches
  python tools/token_bench.py passes [NAME ...]     30 passes of cases of perf/operators.py, for a profiler:
      rocprofv3 --kernel-trace --output-format csv -d DIR -- python3 tools/token_bench.py passes NAME
  python tools/token_bench.py trace DIR             the medians of such a trace, a line a kernel"""
import collections
import csv
import glob
import os
import re
import sys
import time

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

WIDTHS = (16, 40, 64, 100, 128, 200, 256, 384, 512, 520, 777, 1024, 1091, 2048, 2100, 4096, 4099, 4100, 8192, 9000, 12345, 16384)
ROTARY = ((20, 128, 128, False, "bthd"), (20, 128, 64, False, "bthd"), (20, 128, 128, True, "bthd"), (8, 64, 64, False, "bthd"), (1, 64, 64, False, "bthd"), (1, 256, 256, False, "bthd"),
          (20, 128, 128, False, "bhtd"), (4, 64, 64, True, "bhtd"), (12, 80, 40, False, "bthd"), (12, 96, 96, True, "bhtd"), (40, 32, 32, False, "bthd"))
SIZE = 128 << 20


def median(fn, n=12):
    """Seconds of one call, by events around each."""
    import torch
    for _ in range(3):
        fn()
    e = [torch.cuda.Event(enable_timing=True) for _ in range(2 * n)]
    for i in range(n):
        e[2 * i].record()
        fn()
        e[2 * i + 1].record()
    torch.cuda.synchronize()
    return sorted(e[2 * i].elapsed_time(e[2 * i + 1]) for i in range(n))[n // 2] * 1e-3


def norm_rates(D, dt):
    import torch
    from yolopoint_amd import _hip
    l, s, rows = _hip.lib(), _hip.stream_ptr(), SIZE // (D * dt.itemsize)
    x, r, dy, dz = (torch.randn(rows, D, device="cuda").to(dt) for _ in range(4))
    y, z, stats = torch.empty_like(x), torch.empty_like(x), torch.empty(rows, 3, device="cuda")
    w, b, dw, db = torch.ones(D, device="cuda"), torch.zeros(D, device="cuda"), torch.empty(D, device="cuda"), torch.empty(D, device="cuda")
    code = _hip.dtype_code(dt)
    nb = l.yp_layer_norm_bwd_workspace_bytes(rows, D, code)
    ws = torch.empty(nb, dtype=torch.uint8, device="cuda")
    how = dict(rows=rows, D=D, dtype=code, wdtype=_hip.YP_F32, eps=1e-5, x_stride=D, res_stride=D, dy_stride=D, dz_stride=D, weight=w.data_ptr(), bias=b.data_ptr(), stats=stats.data_ptr(),
               seed=1, offset=2, x=x.data_ptr())
    back = dict(how, dy=dy.data_ptr(), dres=y.data_ptr(), dweight=dw.data_ptr(), dbias=db.data_ptr(), workspace=ws.data_ptr(), workspace_bytes=nb)
    calls = ((l.yp_layer_norm_fwd, _hip.YpLayerNormDesc(y=y.data_ptr(), **how), 2, "fwd"), (l.yp_layer_norm_fwd, _hip.YpLayerNormDesc(res=r.data_ptr(), z=z.data_ptr(), y=y.data_ptr(), p=0.1, **how), 4, "fused fwd"),
             (l.yp_layer_norm_bwd, _hip.YpLayerNormDesc(**back), 3, "bwd"), (l.yp_layer_norm_bwd, _hip.YpLayerNormDesc(dz=dz.data_ptr(), dx=z.data_ptr(), p=0.1, **back), 5, "fused bwd"))
    out = []
    for f, d, tensors, name in calls:
        _hip.check(f(d, s))
        t = median(lambda: f(d, s))
        out.append(f"{name} {t * 1e6:7.1f} us {tensors * rows * D * dt.itemsize / t / 1e12:5.2f} TB/s")
    print(f"{str(dt)[6:]:8s} D {D:5d} rows {rows:8d}  " + " | ".join(out), flush=True)


def rates():
    import torch
    from yolopoint_amd import _hip
    from yolopoint_amd.utils import token_ops as ops
    for dt in (torch.bfloat16, torch.float32):
        for D in WIDTHS:
            norm_rates(D, dt)
    l, s = _hip.lib(), _hip.stream_ptr()
    for dt in (torch.bfloat16, torch.float32):
        for n in (SIZE // dt.itemsize, SIZE // dt.itemsize - 3):
            x = torch.randn(n, device="cuda").to(dt)
            r, y = x.clone(), torch.empty_like(x)
            for res, tensors in ((None, 2), (r.data_ptr(), 3)):
                t = median(lambda: l.yp_dropout(x.data_ptr(), res, y.data_ptr(), n, _hip.dtype_code(dt), 0.1, 1, 2, None, s))
                print(f"dropout {str(dt)[6:]:8s} n {n} residual {int(res is not None)}  {t * 1e6:.1f} us {tensors * n * dt.itemsize / t / 1e12:.2f} TB/s", flush=True)
    for dt in (torch.bfloat16, torch.float32):
        for H, D, R, inter, layout in ROTARY:
            T = SIZE // (4 * H * D * dt.itemsize)
            q = torch.randn((4, T, H, D) if layout == "bthd" else (4, H, T, D), device="cuda").to(dt)
            inv, pos = ops.rotary_frequencies(R)[0].cuda(), torch.arange(T, device="cuda")
            with torch.no_grad():
                t = median(lambda: ops.rotary(q, pos, inv, interleaved=inter, layout=layout))
            print(f"rotary {str(dt)[6:]:8s} H {H} D {D} R {R} il {int(inter)} {layout}  {t * 1e6:.1f} us {2 * q.numel() * dt.itemsize / t / 1e12:.2f} TB/s", flush=True)


def copies():
    import torch

    def wall(fn, n):
        for _ in range(3):
            fn()
        torch.cuda.synchronize()
        t = time.perf_counter()
        for _ in range(n):
            fn()
        torch.cuda.synchronize()
        return (time.perf_counter() - t) / n
    for mb in (16, 64, 256, 1024, 4096):
        x = torch.empty(mb << 20, dtype=torch.uint8, device="cuda")
        y = torch.empty_like(x)
        print(f"copy of {mb} MiB: {2 * x.numel() / wall(lambda: y.copy_(x), 20) / 1e12:.2f} TB/s read + written", flush=True)
    a, b = (torch.randn(8192, 8192, device="cuda").bfloat16() for _ in range(2))
    print(f"bf16 product 8192^3: {2 * 8192 ** 3 / wall(lambda: a @ b, 20) / 1e12:.0f} TFLOP/s")


def passes(names):
    import torch
    import perf.operators as cases
    cases.own = True
    for c in cases.listed():
        if names and c["name"] not in names:
            continue
        states = [cases.prepare(dict(c), i) for i in range(3)]
        for i in range(30):
            cases.run(states[i % 3])
        torch.cuda.synchronize()


def trace(folder):
    kinds = collections.OrderedDict()
    for r in csv.DictReader(open(glob.glob(folder + "/**/*kernel_trace.csv", recursive=True)[0])):
        m = re.search(r"(ln_fwd|ln_bwd|ln_columns|dropout|rotary)_kernel(.*)", r["Kernel_Name"])
        if not m:
            continue
        rest = m.group(2)
        kind = "bf16" if "DF16b" in rest else "f16" if "DF16_" in rest else "f32"
        numbers = re.findall(r"Li(\d+)E", rest) or re.findall(r"\b(\d+)\b", rest.split("(")[0])
        flags = re.findall(r"Lb(\d)E", rest) or [str(int(v == "true")) for v in re.findall(r"\b(true|false)\b", rest.split("(")[0])]
        label = f"{m.group(1)}<{kind}"
        if m.group(1) in ("ln_fwd", "ln_bwd"):
            label += f", G={numbers[0]}, E={numbers[1]}" + ", residual" * (flags[0] == "1") + ", dropout" * (flags[1] == "1")
        elif m.group(1) == "dropout":
            label += ", residual" * (flags[0] == "1")
        key = (label + ">", int(r["Grid_Size_X"]) // int(r["Workgroup_Size_X"]), int(r["Workgroup_Size_X"]))
        kinds.setdefault(key, []).append(int(r["End_Timestamp"]) - int(r["Start_Timestamp"]))
    for (label, blocks, threads), v in kinds.items():
        v.sort()
        print(f"  {label:44s} {blocks:6d} workgroups of {threads:4d}  calls {len(v):4d}  median {v[len(v) // 2] / 1e3:8.2f} us  min {v[0] / 1e3:8.2f}")


if __name__ == "__main__":
    what = sys.argv[1] if len(sys.argv) > 1 else ""
    if what == "rates":
        rates()
    elif what == "copies":
        copies()
    elif what == "passes":
        passes(sys.argv[2:])
    elif what == "trace" and len(sys.argv) > 2:
        trace(sys.argv[2])
    else:
        sys.exit(__doc__)
