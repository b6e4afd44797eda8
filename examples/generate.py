"""Trains a small Mesh GPT on modular equations, then scores and generates
answers over its 8-bit key/value cache.

    python examples/generate.py [--modulus 23] [--steps 400]
"""

import argparse
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import numpy as np  # noqa: E402

from grokking_abmod_b200 import CachedGpt, GptConfig, MeshGpt  # noqa: E402
from grokking_abmod_b200.data import EquationDataset, EquationSampler  # noqa: E402


def main():
    parser = argparse.ArgumentParser()
    parser.add_argument("--modulus", type=int, default=23)
    parser.add_argument("--steps", type=int, default=400)
    args = parser.parse_args()

    data = EquationDataset(args.modulus, "add", 0.8, 1)
    config = GptConfig(vocab_size=data.vocab_size, context=8, width=128, heads=4, layers=2)
    model = MeshGpt(0, config, 7)
    sampler = EquationSampler(len(data.training), 3)
    for step in range(args.steps):
        x, y = data.batch(False, sampler.sample(min(512, len(data.training))))
        loss = model.train_batch(x, y, 4, 0.01, 0.1)
        if step % 100 == 99:
            print(f"step {step + 1}: loss {loss:.4f}")

    x, y = data.batch(False, np.arange(min(64, len(data.training))))
    prompts, answers = x.reshape(-1, 4).tolist(), y.reshape(-1, 4)[:, 3].astype(np.int64)
    scored = CachedGpt(model, len(prompts)).score(prompts, answers, top=3)
    print(f"log-probability of the right answers: mean {scored.logprob.mean():.4f}, worst {scored.logprob.min():.4f};"
          f" entropy {scored.entropy.mean():.4f} nats")
    print("first prompt's alternatives:", list(zip(scored.top_index[0].tolist(), scored.top_logprob[0].tolist())))
    first = CachedGpt(model, len(prompts)).generate(prompts, 1)[0]
    print(f"greedy answers right: {(first.top_index[:, 0].cpu().numpy() == answers).mean():.1%}")


if __name__ == "__main__":
    main()
