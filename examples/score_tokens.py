"""Score given next tokens with an int8 head: hidden rows -> TInt8ConnectedLayer -> logits ->
TTokenLogprobsLayer (log probability of each given token, entropy, the most probable tokens), then one
training step's gradient with respect to the logits. Weights and hidden rows are random.

    python examples/score_tokens.py [--rows 64] [--hidden 1024] [--vocab 32000] [--top 5]
"""
import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from tensorium_b200 import Context
from tensorium_b200.layers import TInt8ConnectedLayer, TNNetState, TTokenLogprobsLayer


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("rows", 64), ("hidden", 1024), ("vocab", 32000), ("top", 5), ("seed", 0)):
        ap.add_argument(f"--{name}", type=int, default=value)
    a = ap.parse_args(argv)
    g = torch.Generator(device="cuda").manual_seed(a.seed)
    hidden = torch.randn(a.rows, a.hidden, device="cuda", generator=g).to(torch.bfloat16)
    weights = torch.randn(a.vocab, a.hidden, device="cuda", generator=g) * a.hidden ** -0.5
    given = torch.randint(a.vocab, (a.rows,), device="cuda", generator=g)
    with Context(0) as ctx:
        head = TInt8ConnectedLayer(a.hidden, a.vocab, weights=weights).bind(ctx)
        scorer = TTokenLogprobsLayer(top=a.top).bind(ctx)
        logits = head.forward(TNNetState(hidden))
        r = scorer.forward(TNNetState(logits), given)
        # the loss is the mean of -logprob
        grad = scorer.backward(TNNetState(logits), given, torch.full_like(r.logprobs, -1 / a.rows))
        ctx.sync()
    print(f"mean log probability of the given tokens {r.logprobs.mean():.4f}, mean entropy {r.entropy.mean():.4f}")
    for i in range(min(4, a.rows)):
        tops = ", ".join(f"{t}: {p:.3f}" for t, p in zip(r.top_tokens[i].tolist(), r.top_logprobs[i].exp().tolist()))
        print(f"row {i}: token {given[i].item()} at {r.logprobs[i].exp():.2e}; most probable {tops}")
    print(f"gradient norm {grad.float().norm():.4e}")
    return hidden, weights, given, r, grad


if __name__ == "__main__":
    main()
