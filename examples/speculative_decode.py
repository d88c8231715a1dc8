"""Speculative decoding with drafts looked up in the text so far.

A random-init MXFP4 decoder (7B widths by default, fewer layers) on a
block-scaled fp8 cache answers ragged prompts twice: one token a step, then with
drafts that followed the last occurrence of the text's last two tokens.  Every
step appends and attends the last token and the drafts, then verifies the drafts.
Random weights repeat nothing, so the layers' norms are turned down and the
output head is the embedding with tokens moved on by one within groups of 32: the
model counts, and its texts have repetitions to look up.

    python examples/speculative_decode.py [--layers 4] [--batch 4] [--drafts 4] [--tokens 256]
                                          [--window 0] [--sinks 0] [--temperature 1]
"""
import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gfx1201-tuning-log_b200"))
import decoder  # noqa: E402
import spec_decoder  # noqa: E402


def look_up(text, k):
    """k drafts: what followed the last earlier occurrence of the text's last two
    tokens (of the last one, where there is none), repeated past the end."""
    for n in (2, 1):
        for i in range(len(text) - n - 1, -1, -1):
            if text[i:i + n] == text[-n:]:
                found = text[i + n:i + n + k]
                return found + [found[-1]] * (k - len(found))
    return [text[-1]] * k


def answer(model, prompts, tokens, heat, g, drafts):
    """New tokens, steps and seconds of answers of at least `tokens` tokens each."""
    first = model.prompt(prompts, heat, g)
    texts = [p.tolist() + [t] for p, t in zip(prompts, first.tolist())]
    torch.cuda.synchronize()
    begin, steps = time.perf_counter(), 0
    while min(len(t) - len(p) for t, p in zip(texts, prompts)) < tokens:
        guess = torch.tensor([look_up(t, drafts) if drafts else [] for t in texts], dtype=torch.int64)
        out, accepted = model.verify_step(guess.view(len(texts), drafts).to(model.dev), heat, generator=g)
        for text, row, n in zip(texts, out.tolist(), accepted.tolist()):
            text += row[:n + 1]
        steps += 1
    return sum(len(t) - len(p) for t, p in zip(texts, prompts)), steps, time.perf_counter() - begin


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("layers", 4), ("batch", 4), ("drafts", 4), ("tokens", 256), ("window", 0), ("sinks", 0),
                        ("prompt", 512), ("vocab", 128256)):
        ap.add_argument(f"--{name}", type=int, default=value)
    ap.add_argument("--temperature", type=float, default=1.0)
    a = ap.parse_args()
    dev = torch.device("cuda", 0)
    g = torch.Generator(device=dev).manual_seed(0)
    # a sequence that runs ahead of the slowest takes up to drafts + 1 tokens a step
    model = spec_decoder.SpeculativeDecoder(decoder.DecoderConfig(layers=a.layers, vocab=a.vocab), dev, a.batch,
                                            a.prompt + (a.tokens + 1) * (a.drafts + 1), window=a.window, sinks=a.sinks)
    for layer in model.layers:
        layer["in_norm"].mul_(0.001)
        layer["post_norm"].mul_(0.001)
    before = torch.arange(a.vocab, device=dev)
    before = before // 32 * 32 + (before - 1) % 32
    model.lm_head = 0.02 * model.embed[before.clamp_max(a.vocab - 1)]
    heat = torch.full((a.batch,), a.temperature, device=dev)
    prompts = [torch.randint(0, a.vocab, (a.prompt - 37 * i % (a.prompt // 2),), device=dev, generator=g)
               for i in range(a.batch)]
    for drafts in (0, a.drafts):
        answer(model, prompts, 2, heat, g, drafts)  # warm up
        new, steps, seconds = answer(model, prompts, a.tokens, heat, g, drafts)
        print(f"{drafts} drafts: {new} tokens of {a.batch} sequences in {steps} steps, {new / seconds:.0f} tok/s")


if __name__ == "__main__":
    main()
