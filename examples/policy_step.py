"""One policy-gradient step of a small decoder whose entropy bonus is the series variable.

The loss of a sampled batch is

    loss(t) = -mean(advantage * log p(token)) - (bonus + t) * mean(entropy),

with t the series variable: after the step every parameter is a power series in t, whose first plane
past the value says how the trained weights answer to the entropy bonus.  The model uses the token
operators together: heads normalised and rotated in one pass in front of attention, dropout added to
the residual, log probabilities and entropy of the sampled tokens, and a decoding step that asks for
the best alternatives.

    python examples/policy_step.py
"""

import math
import pathlib
import sys

import torch
import torch.nn.functional as F

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parents[1] / "poly-tensors_b200"))

from polytensors_b200 import PolyTensor  # noqa: E402


class Decoder:
    """Pre-norm decoder with per-head query / key norms and rotary positions."""

    def __init__(self, vocab=512, width=128, heads=4, layers=2, degree=2, positions=256, seed=0, device="cuda"):
        self.width, self.heads, self.layers, self.degree = width, heads, layers, degree
        g = torch.Generator().manual_seed(seed)

        def weight(*shape):
            value = torch.randn(*shape, generator=g) * 0.02 if len(shape) > 1 else torch.ones(*shape)
            return torch.nn.Parameter(PolyTensor((value.to(device),), degree=degree))

        head = width // heads
        self.p = {"emb": weight(vocab, width), "norm": weight(width), "out": weight(vocab, width)}
        for i in range(layers):
            self.p |= {f"norm1.{i}": weight(width), f"norm2.{i}": weight(width), f"up.{i}": weight(4 * width, width),
                       f"down.{i}": weight(width, 4 * width), f"qn.{i}": weight(head), f"kn.{i}": weight(head)}
            self.p |= {f"{name}.{i}": weight(width, width) for name in "qkvo"}
        angle = torch.arange(positions, dtype=torch.float64)[:, None] \
            * 10000.0 ** (-torch.arange(0, head, 2, dtype=torch.float64) / head)
        self.cos, self.sin = angle.cos().float().to(device), angle.sin().float().to(device)

    def logits(self, ids, dropout=0.0, seed=0):
        B, T = ids.shape
        H, D = self.heads, self.width // self.heads
        p, x = self.p, F.embedding(ids, self.p["emb"])
        for i in range(self.layers):
            h = F.rms_norm(x, (self.width,), p[f"norm1.{i}"])
            q, k, v = (F.linear(h, p[f"{name}.{i}"]).view(B, T, H, D) for name in "qkv")
            q, k = PolyTensor.qk_norm_rope(q, k, p[f"qn.{i}"], p[f"kn.{i}"], self.cos, self.sin)
            a = F.scaled_dot_product_attention(q, k, v.transpose(1, 2), is_causal=True)
            a = F.linear(a.transpose(1, 2).reshape(B, T, self.width), p[f"o.{i}"])
            x = PolyTensor.dropout(a, dropout, seed=seed, offset=2 * i, residual=x)
            h = F.gelu(F.linear(F.rms_norm(x, (self.width,), p[f"norm2.{i}"]), p[f"up.{i}"]))
            x = PolyTensor.dropout(F.linear(h, p[f"down.{i}"]), dropout, seed=seed, offset=2 * i + 1, residual=x)
        return F.linear(F.rms_norm(x, (self.width,), p["norm"]), p["out"])


def policy_step(model, ids, advantage, bonus=0.01, lr=0.1, dropout=0.1, seed=1):
    """One SGD step on sampled sequences ``ids`` (B, T + 1) with ``advantage`` (B, T); the loss series."""
    params = list(model.p.values())
    optimizer = torch.optim.SGD(params, lr=lr, foreach=False)
    t = PolyTensor((torch.tensor(0.0, device=ids.device), 1.0), degree=model.degree)
    with PolyTensor.plain_range(), PolyTensor.retain_wrappers():
        got = PolyTensor.token_log_probs(model.logits(ids[:, :-1], dropout, seed), ids[:, 1:])
        loss = -(advantage * got.log_probs).mean() - (bonus + t) * got.entropy.mean()
        loss.backward()
        optimizer.step()
    return [c.item() for c in loss.coeffs]


@torch.no_grad()
def next_tokens(model, ids, top=5, temperature=1.0):
    """The best next tokens of each sequence with their log probabilities (constant plane)."""
    with PolyTensor.plain_range():
        last = model.logits(ids)[:, -1]
        greedy = torch.zeros(ids.shape[0], dtype=torch.int64, device=ids.device)
        got = PolyTensor.token_log_probs(last.value, greedy, top=top, temperature=temperature)
    return got.top_tokens, got.top_log_probs


def main():
    torch.manual_seed(0)
    model = Decoder()
    ids = torch.randint(0, 512, (4, 65), device="cuda")
    advantage = torch.randn(4, 64, device="cuda")
    for step in range(3):
        loss = policy_step(model, ids, advantage, seed=step)
        print(f"step {step}: loss series {', '.join(f'{c:.5f}' for c in loss)}")
    tokens, log_probs = next_tokens(model, ids[:, :-1])
    print("best next tokens of the first sequence:", tokens[0].tolist(),
          [round(math.exp(v), 4) for v in log_probs[0].tolist()])
    answer = model.p["out"].coeffs[1]
    print(f"output weights answer to the entropy bonus with norm {answer.norm().item():.4g}")


if __name__ == "__main__":
    main()
