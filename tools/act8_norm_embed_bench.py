"""Times of the 8-bit checkpoint, RMS norm and scaled-embedding calls over widths and token counts (HIP events around
back-to-back calls, so the smallest are launch-bound).
    python tools/act8_norm_embed_bench.py"""
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from bifold_amd.hip import lib as L  # noqa: E402
from bifold_amd.hip import ops  # noqa: E402


def us(f, n=60):
    for _ in range(8):
        f()
    torch.cuda.synchronize()
    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    a.record()
    for _ in range(n):
        f()
    b.record()
    torch.cuda.synchronize()
    return a.elapsed_time(b) / n * 1e3


def line(what, t, nbytes):
    print(f"{what:52s} {t:8.1f} us  {nbytes / t / 1e6:5.2f} TB/s", flush=True)


for rows, cols, dt in ((36928, 4096, torch.float16), (20000, 1155, torch.bfloat16), (73728, 768, torch.float32)):
    x = torch.randn(rows, cols, device="cuda").to(dt)
    m, e = x.numel(), x.element_size()
    kept = ops.act8_pack(x)
    line(f"act8_pack {rows}x{cols} {dt}", us(lambda: ops.act8_pack(x)), m * (e + 1.03))
    line("act8_unpack", us(lambda: ops.act8_unpack(kept, dt)), m * (e + 1.03))
    line("act8_gelu_fwd (tanh)", us(lambda: ops.act8_gelu_fwd(x, L.ACT_TANH_GELU)), m * (2 * e + 1.03))
    line("act8_gelu_bwd (tanh)", us(lambda: ops.act8_gelu_bwd(x, kept, L.ACT_TANH_GELU)), m * (2 * e + 1.03))
for rows, cols in ((1, 4096), (300, 4096), (2100, 1100), (20000, 1155), (36928, 1024), (40000, 1536), (16384, 2048), (9000, 4096),
                   (4096, 8192), (3000, 12288), (2000, 16384), (2000, 20000)):
    x = torch.randn(rows, cols, device="cuda").half()
    g, dg, delta = torch.ones(cols, device="cuda"), torch.empty(cols, device="cuda"), torch.randn_like(x)
    _, r, kept = ops.rmsnorm_fwd(x, g, torch.float16, save_stats=True, checkpoint=True)
    line(f"rmsnorm_fwd {rows}x{cols} fp16 + delta", us(lambda: ops.rmsnorm_fwd(x, g, x.dtype, delta=delta, write_x=False)),
         x.numel() * 6)
    line("rmsnorm_fwd_fp8", us(lambda: ops.rmsnorm_fwd_fp8(x, g, delta=delta, write_x=False)), x.numel() * 5)
    line("rmsnorm_bwd from the checkpoint, dres", us(lambda: ops.rmsnorm_bwd(delta, kept, g, r, dg, dres=x)), x.numel() * 7.03)
gen = torch.Generator().manual_seed(0)
for n in (64, 512, 513, 2048, 2049, 8192, 131072):
    for kind, share in (("mixed", 0.0), ("half one token", 0.5), ("one token", 1.0)):
        ids = torch.randint(0, 32000, (n,), generator=gen)
        ids[:int(n * share)] = 7
        ids, dy = ids.int().cuda(), torch.randn(n, 1024, device="cuda")
        grad = torch.zeros(32000, 1024, device="cuda")
        a = us(lambda: ops.embed_scaled_bwd(dy, ids, 32000, 1.0, out=grad, accumulate=True))
        d = us(lambda: ops.embed_scaled_bwd(dy, ids, 32000, 1.0, out=grad))
        print(f"embed_scaled_bwd {n}x1024 fp32, {kind:15s} added {a:7.1f} us, whole table {d:7.1f} us", flush=True)
