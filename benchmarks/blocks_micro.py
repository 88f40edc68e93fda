"""The block-scaled 8-bit operators alone: GPU time of each call (captured into a graph, so that the host's part is out of it), at the sizes the
acoustic model and its streams give them.  python benchmarks/blocks_micro.py [--once]   (--once: each call twice, for a profiler)"""
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import torch  # noqa: E402

from stt_amd import blocks  # noqa: E402

E4M3 = torch.float8_e4m3fn


def timed(name, f, reps, note):
    f()
    if "--once" in sys.argv:
        f()
        torch.cuda.synchronize()
        return
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for _ in range(reps):
            f()
    g.replay()
    times = []
    for _ in range(9):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        g.replay()
        b.record()
        b.synchronize()
        times.append(a.elapsed_time(b) * 1e3 / reps)
    us = sorted(times)[4]
    print("%-44s %9.2f us  %s" % (name, us, note(us)), flush=True)


def main():
    act = lambda m, k: (torch.randn(m, k, device="cuda") * torch.exp(1.5 * torch.randn(m, 1, device="cuda"))).clamp_(0, 20)
    for m, k, t in ((16, 494, torch.float32), (32000, 2048, torch.float16), (32000, 2048, torch.float32)):
        x = act(m, k).to(t)
        timed("quantise %d x %d %s" % (m, k, t), lambda: blocks.quantize_blocks(x), 20, lambda us: "%7.0f GB/s" % (m * k * (x.element_size() + 1) / us / 1e3))
    for t in (torch.float32, torch.float16):
        w = torch.randn(8192, 2048, device="cuda").to(t)
        timed("quantise tiles 8192 x 2048 %s" % t, lambda: blocks.quantize_blocks(w, 128), 20, lambda us: "%7.0f GB/s" % (w.numel() * (w.element_size() + 1) / us / 1e3))
    b = blocks.quantize_blocks(act(32000, 2048))
    for t, size in ((torch.bfloat16, 2), (torch.float32, 4)):
        timed("read back 32000 x 2048 to %s" % t, lambda: blocks.dequantize_blocks(b, t), 20, lambda us: "%7.0f GB/s" % (32000 * 2048 * (1 + size) / us / 1e3))
    wb = blocks.quantize_blocks(w, 128)
    timed("read back tiles 8192 x 2048 to f16", lambda: blocks.dequantize_blocks(wb, torch.float16), 20, lambda us: "%7.0f GB/s" % (8192 * 2048 * 3 / us / 1e3))
    for m, k, n, src, dst in ((1, 2048, 2048, "f16", "f16"), (16, 494, 2048, "f32", "blocks"), (16, 2048, 2048, "blocks", "blocks"), (16, 2048, 8192, "blocks", "f32"),
                              (64, 2048, 2048, "f16", "f16"), (256, 2048, 2048, "blocks", "f16"), (512, 2048, 2048, "blocks", "f16"), (512, 2048, 8192, "blocks", "f32"),
                              (1024, 2048, 2048, "blocks", "f16"), (2048, 2048, 2048, "blocks", "f16"), (1009, 2048, 29, "bf16", "f32"), (2048, 2048, 8192, "blocks", "f32"),
                              (6144, 2048, 2048, "blocks", "blocks"), (6144, 2048, 8192, "blocks", "f16"), (32000, 2048, 8192, "blocks", "f32")):
        types = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "blocks": E4M3}
        x = act(m, k)
        x = blocks.quantize_blocks(x) if src == "blocks" else x.to(types[src])
        w = blocks.quantize_blocks(torch.randn(n, k, device="cuda") / k ** 0.5, 128)
        c = torch.randn(n, device="cuda")
        timed("dense %d x %d -> %d, %s -> %s" % (m, k, n, src, dst), lambda: blocks.dense_blocks(x, w, c, relu_clip=20.0 if dst == "blocks" else None, dtype=types[dst]),
              20, lambda us: "%7.1f TFLOP/s" % (2.0 * m * k * n / us / 1e6))


if __name__ == "__main__":
    main()
