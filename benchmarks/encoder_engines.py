"""The embedding model's two engines against each other: a 12-layer, 768-wide MPNet with 12 heads, a feed-forward of 2048 and random
weights (written to a temporary directory), through MPNetEmbedder.embed_device(), tokenisation included.

    python3 benchmarks/encoder_engines.py [--out FILE]

One JSON line per precision and engine: milliseconds for one text of 14 tokens, 2048 texts of 5 to 32 tokens, 256 texts of 302 tokens
(batches of 64, the embedder's default), and the mean 2-norm of the vectors' difference from the transformers engine in fp32."""
import argparse
import json
import os
import random
import sys
import tempfile
import time

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import torch  # noqa: E402
from transformers import MPNetConfig, MPNetModel, MPNetTokenizer  # noqa: E402

from vectordb_amd.embedders import MPNetEmbedder  # noqa: E402

WORDS = [f"w{i}" for i in range(200)]


def write_model(d):
    with open(os.path.join(d, "vocab.txt"), "w") as f:
        f.write("\n".join(["<s>", "<pad>", "</s>", "<unk>", "<mask>", *WORDS]) + "\n")
    MPNetTokenizer(os.path.join(d, "vocab.txt")).save_pretrained(d)
    torch.manual_seed(0)
    MPNetModel(MPNetConfig(vocab_size=len(WORDS) + 5, hidden_size=768, num_hidden_layers=12, num_attention_heads=12, intermediate_size=2048,
                           max_position_embeddings=514)).save_pretrained(d)


def ms(call, times):
    for _ in range(3):
        call()
    torch.cuda.synchronize()
    t = time.perf_counter()
    for _ in range(times):
        call()
    torch.cuda.synchronize()
    return (time.perf_counter() - t) / times * 1e3


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--out")
    args = ap.parse_args()
    rng = random.Random(0)

    def text(n):
        return " ".join(rng.choice(WORDS) for _ in range(n))
    sets = {"one_text_14": ([text(12)], 50), "2048_texts_5_to_32": ([text(rng.randint(3, 30)) for _ in range(2048)], 3),
            "256_texts_302": ([text(300) for _ in range(256)], 3)}
    lines = []
    with tempfile.TemporaryDirectory() as d:
        write_model(d)
        plain = None
        for amp in (None, "bf16", "fp16"):
            for engine in ("transformers", "hip"):
                e = MPNetEmbedder(d, device="cuda:0", autocast=amp, engine=engine)
                some = e.embed_device(sets["2048_texts_5_to_32"][0][:64])
                plain = some if plain is None else plain
                line = {"precision": amp or "fp32", "engine": engine, "error": float(f"{float((some - plain).norm(dim=1).mean()):.3g}")}
                line.update({n: round(ms(lambda: e.embed_device(texts), k), 3) for n, (texts, k) in sets.items()})
                lines.append(line)
                print(json.dumps(line), flush=True)
    if args.out:
        with open(args.out, "w") as f:
            f.write("".join(json.dumps(x) + "\n" for x in lines))


if __name__ == "__main__":
    main()
