#!/usr/bin/env python3
"""Micro-benchmark of the layer-norm and dropout entry points: HIP-event time of back-to-back calls on alternating
buffers and the bytes they move (forward x -> y, backward x, dy -> dx; residual form x, res -> s, y and dy, ds, s -> dx,
dres), beside a device copy of the same size."""
import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
for p in (ROOT, os.path.join(ROOT, "soft-intro-vae-for-3d-mri_amd")):
    sys.path.insert(0, p)
import torch  # noqa: E402
import siv.backend as sb  # noqa: E402

TYPES = {"fp32": (torch.float32, 0), "bf16": (torch.bfloat16, 1), "fp16": (torch.float16, 2)}
ROWS = [(4915200, 64, "fp32"), (614400, 128, "fp32"), (614400, 128, "bf16"), (76800, 256, "bf16"), (9600, 256, "bf16"),
        (20000, 1024, "bf16"), (16384, 2048, "fp32"), (8192, 4096, "fp32"), (8192, 8192, "bf16"), (2000, 16384, "bf16"),
        (300, 100000, "fp32"), (8, 38400, "fp16"), (100000, 601, "bf16"), (1050, 601, "bf16"), (200000, 33, "fp32"),
        (4, 600, "fp32")]
FLAT = [(314572800, "bf16"), (78643200, "fp32"), (78643201, "fp32"), (19660800, "bf16"),
        (50331648, "bf16"), (100663296, "bf16"), (787101, "fp16"), (9600, "fp32")]


def timeit(fns, reps):
    for f in fns:
        f()
    torch.cuda.synchronize()
    times = []
    for _ in range(5):
        e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        e0.record()
        for i in range(reps):
            fns[i % len(fns)]()
        e1.record()
        torch.cuda.synchronize()
        times.append(e0.elapsed_time(e1) / reps)
    return sorted(times)[2]


def report(name, fns, nbytes):
    ms = timeit(fns, max(4, min(200, int(3e9 / nbytes))))
    print(f"{name:34s} {ms * 1e3:9.1f} us  {nbytes / ms / 1e9:6.2f} TB/s", flush=True)


def main():
    B = sb.get_backend()
    L, st = B.lib, torch.cuda.current_stream().cuda_stream
    ptr = lambda t: t.data_ptr()
    for R, C, name in ROWS:
        dt, ty = TYPES[name]
        n = R * C
        size = n * dt.itemsize
        sets = [[torch.randn(n, device="cuda").to(dt) for _ in range(3)] +
                [torch.empty(n, device="cuda", dtype=dt) for _ in range(2)] for _ in range(2)]
        w, b, dw, db = (torch.ones(C, device="cuda") for _ in range(4))
        nb = max(sb._norm_ws_bytes(R, C, ty, 0), sb._norm_ws_bytes(R, C, ty, 1), 16)
        ws = torch.empty(nb, dtype=torch.uint8, device="cuda")
        tag = f"{R} x {C} {name}"
        report(f"norm fwd {tag}", [lambda s=s: L.siv_layer_norm_fwd(
            ptr(s[0]), C, ptr(w), ptr(b), 0, 1e-5, ptr(s[3]), ty, R, C, ptr(ws), nb, st) for s in sets], 2 * size)
        report(f"norm bwd {tag}", [lambda s=s: L.siv_layer_norm_bwd(
            ptr(s[1]), C, ptr(s[0]), C, ptr(w), 0, 1e-5, ptr(s[3]), ptr(dw), ptr(db), 0, ty, R, C, ptr(ws), nb, st)
            for s in sets], 3 * size)
        report(f"add+norm fwd {tag}", [lambda s=s: L.siv_add_layer_norm_fwd(
            ptr(s[0]), ptr(s[1]), None, 5, 7, None, 0.25, ptr(w), ptr(b), 0, 1e-5, ptr(s[3]), ptr(s[4]), ty, R, C, ptr(ws),
            nb, st) for s in sets], 4 * size)
        report(f"add+norm bwd {tag}", [lambda s=s: L.siv_add_layer_norm_bwd(
            ptr(s[0]), ptr(s[1]), ptr(s[2]), None, 5, 7, None, 0.25, ptr(w), 0, 1e-5, ptr(s[3]), ptr(s[4]), ptr(dw), ptr(db),
            0, ty, R, C, ptr(ws), nb, st) for s in sets], 5 * size)
        del sets, ws
        torch.cuda.empty_cache()
    for n, name in FLAT:
        dt, ty = TYPES[name]
        size = n * dt.itemsize
        sets = [[torch.randn(n, device="cuda").to(dt) for _ in range(2)] + [torch.empty(n, device="cuda", dtype=dt)]
                for _ in range(2)]
        report(f"dropout {n} {name}", [lambda s=s: L.siv_dropout_fwd(
            ptr(s[0]), None, None, 5, 7, None, 0.35, 1.0, ptr(s[2]), ty, n, st) for s in sets], 2 * size)
        report(f"dropout+res {n} {name}", [lambda s=s: L.siv_dropout_fwd(
            ptr(s[0]), ptr(s[1]), None, 5, 7, None, 0.35, 1.0, ptr(s[2]), ty, n, st) for s in sets], 3 * size)
        report(f"copy {n} {name}", [lambda s=s: s[2].copy_(s[0]) for s in sets], 2 * size)
        del sets
        torch.cuda.empty_cache()


if __name__ == "__main__":
    main()
