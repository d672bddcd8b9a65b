"""The encoder operators' forms on the GPU alone: ten calls captured into a HIP graph and replayed, inputs as they lie in the caches after
the call before.

    python3 benchmarks/encoder_ops.py [--out FILE]

One JSON line per form and type: microseconds a call, and its floor = max(bytes / 4.9 TB/s, operations / rate) with the rates that a 2 GiB copy
and an 8192^3 library product reach on an MI355X (1.44 PFLOP/s bf16, 1.50 fp16, 153 TFLOP/s fp32).  "backward" is the gradient's part: a
pass with all gradients less the forward pass that keeps what they need."""
import argparse
import json
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import torch  # noqa: E402

from vectordb_amd import ops  # noqa: E402

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
RATE = {"fp32": 153e12, "bf16": 1.44e15, "fp16": 1.50e15}
COPY = 4.9e12


def replayed(step, calls=10, turns=5):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(calls):
            step()
    best = []
    for _ in range(turns + 2):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        graph.replay()
        b.record()
        b.synchronize()
        best.append(a.elapsed_time(b) * 1e3 / calls)
    return sorted(best[2:])[turns // 2]


def linear_forms():
    for m, n, k, act, res in ((14, 2304, 768, "none", False), (480, 768, 768, "none", True), (1999, 1536, 384, "gelu", False), (6144, 768, 768, "none", True),
                              (8192, 1536, 768, "gelu", False), (49152, 2304, 768, "none", False), (8192, 1535, 767, "gelu", False)):
        yield f"linear {m} x {n} from {k}{'' if act == 'none' else ' ' + act}{' residual' if res else ''}", m, n, k, act, res


def attention_forms():
    g = torch.Generator().manual_seed(0)
    ragged = torch.randint(3, 65, (512,), generator=g).tolist()
    train = torch.randint(16, 385, (64,), generator=g).tolist()
    for name, lengths, heads, d in (("14 tokens", [14], 12, 64), ("512 texts of 3 to 64", ragged, 12, 32), ("16 x 384", [384] * 16, 12, 64), ("64 texts of 16 to 384", train, 12, 64),
                                    ("4095 + 2564 + 1033", [4095, 2564, 1033], 12, 64), ("64 texts of 16 to 384", train, 6, 128), ("64 texts of 16 to 384", train, 12, 24),
                                    ("64 texts of 16 to 384", train, 12, 80), ("64 texts of 16 to 384", train, 12, 96)):
        yield f"attention {name}, {heads} heads of {d}", lengths, heads, d


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--out")
    args = ap.parse_args()
    lines = []

    def report(form, dtype, what, us, flops, nbytes):
        floor = max(nbytes / COPY, flops / RATE[dtype]) * 1e6
        lines.append({"form": form, "type": dtype, "pass": what, "us": round(us, 1), "floor_us": round(floor, 2), "tflops": round(flops / us * 1e-6, 1), "gbs": round(nbytes / us * 1e-3)})
        print(json.dumps(lines[-1]), flush=True)

    def both(form, dtype, call, leaves, dy, flops, nbytes, back_flops, back_bytes):
        with torch.no_grad():
            report(form, dtype, "forward", replayed(call), flops, nbytes)

        def step(grads):
            own = [t.detach().requires_grad_() for t in leaves]
            y = call(*own)
            return torch.autograd.grad(y, own, dy) if grads else y
        report(form, dtype, "backward", replayed(lambda: step(True)) - replayed(lambda: step(False)), back_flops, back_bytes)

    for dtype, t in TYPES.items():
        size = t.itemsize
        for form, m, n, k, act, res in linear_forms():
            x, w, b = torch.randn(m, k, device="cuda").to(t), (torch.randn(n, k, device="cuda") * k ** -0.5).to(t), torch.randn(n, device="cuda").to(t)
            r, dy = (torch.randn(m, n, device="cuda").to(t) if res else None), torch.randn(m, n, device="cuda").to(t)
            io = (m * k + n * k + n + m * n * (2 if res else 1)) * size
            both(form, dtype, lambda x=x, w=w, b=b: ops.linear(x, w, b, act, r), [x, w, b], dy, 2.0 * m * n * k, io, 4.0 * m * n * k, (2 * m * k + 2 * n * k + m * n * (2 if act != "none" else 1)) * size)
        for form, lengths, heads, d in attention_forms():
            total, squares = sum(lengths), sum(v * v for v in lengths)
            off = torch.tensor([0, *torch.tensor(lengths).cumsum(0).tolist()], device="cuda")
            qkv, table, dy = torch.randn(total, 3, heads, d, device="cuda").to(t), torch.randn(32, heads, device="cuda").to(t), torch.randn(total, heads, d, device="cuda").to(t)
            both(form, dtype, lambda q=qkv, b=table: ops.bucketed_attention(q, b, off), [qkv, table], dy, 4.0 * squares * heads * d, 4 * total * heads * d * size,
                 10.0 * squares * heads * d, 8 * total * heads * d * size)
        for count, longest in ((1, 14), (1024, 128)):
            lengths = [3 + i * (longest - 3) // max(1, count - 1) for i in range(count)] if count > 1 else [longest]
            total = sum(lengths)
            off = torch.tensor([0, *torch.tensor(lengths).cumsum(0).tolist()], device="cuda")
            h, dy = torch.randn(total, 768, device="cuda").to(t), torch.randn(count, 768, device="cuda")
            rows = total * 768 * size + count * 768 * 4
            both(f"mean pool {count} texts, {total} rows of 768", dtype, lambda h=h: ops.mean_pool(h, off), [h], dy, total * 768.0, rows, total * 768.0, rows)
    if args.out:
        with open(args.out, "w") as f:
            f.write("".join(json.dumps(x) + "\n" for x in lines))


if __name__ == "__main__":
    main()
