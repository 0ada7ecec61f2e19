"""Trains a small language model of expert blocks, then decodes a few tokens with it.

    python -m examples.train_experts [--steps 60] [--device cuda|cpu] [--precision fp32|bf16|fp8]

A block is ``x + combine(down(gelu(up(dispatch(layer_norm(x))))))``: the package's layer norm, a router that
chooses ``top_k`` of the experts for each token, the rows' way to them, their products, and the way back.  The
loss is ``causal_lm_loss``, the optimizer ``AdamBridge`` (on the GPU; on the CPU, where its kernels do not
run, torch's AdamW).  Nothing in a step waits for the device: the losses are read when the steps are done.
"""

import argparse

import torch
import torch.nn.functional as F

import adambridge_amd as ab


class ExpertBlock(torch.nn.Module):
    """Layer norm, ``experts`` MLPs of hidden -> inter -> hidden of which each token takes ``top_k``, a residual."""

    def __init__(self, hidden: int, inter: int, experts: int, top_k: int):
        super().__init__()
        self.top_k = top_k
        self.norm = torch.nn.LayerNorm(hidden)
        self.router = torch.nn.Linear(hidden, experts, bias=False)
        self.up = torch.nn.Parameter(torch.randn(experts, inter, hidden) * hidden ** -0.5)
        self.down = torch.nn.Parameter(torch.randn(experts, hidden, inter) * inter ** -0.5)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        flat = x.reshape(-1, x.shape[-1])
        h = ab.layer_norm(flat, self.norm.weight, self.norm.bias, self.norm.eps)
        r = ab.route(self.router(h), self.top_k)
        rows = F.gelu(ab.expert_mm(ab.dispatch(h, r), self.up, r.ends))
        return (flat + ab.combine(ab.expert_mm(rows, self.down, r.ends), r)).view(x.shape)


class Model(torch.nn.Module):
    """Embedding, expert blocks (with a causal mean of the tokens before, in place of attention), head."""

    def __init__(self, vocab: int = 512, hidden: int = 128, inter: int = 256, experts: int = 8, top_k: int = 2, layers: int = 2):
        super().__init__()
        self.embed = torch.nn.Embedding(vocab, hidden)
        self.blocks = torch.nn.ModuleList(ExpertBlock(hidden, inter, experts, top_k) for _ in range(layers))
        self.norm = torch.nn.LayerNorm(hidden)
        self.head = torch.nn.Linear(hidden, vocab, bias=False)

    def forward(self, ids: torch.Tensor) -> torch.Tensor:
        """Hidden states of ``ids`` [batch, seq], ready for the head."""
        x = self.embed(ids)
        count = torch.arange(1, ids.shape[1] + 1, device=ids.device)[:, None]
        for block in self.blocks:
            x = block(x + (x.float().cumsum(1) / count).to(x.dtype))
        return ab.layer_norm(x, self.norm.weight, self.norm.bias, self.norm.eps)


def fit(model: Model, opt: torch.optim.Optimizer, ids: torch.Tensor, steps: int, batch: int, seq: int) -> list[torch.Tensor]:
    """``steps`` steps on windows of ``ids``; their losses, on the device."""
    losses = []
    for step in range(steps):
        starts = torch.randint(0, 16, (batch,)).tolist()
        x = torch.stack([ids[s:s + seq] for s in starts])
        loss = ab.causal_lm_loss(model(x), model.head, x)
        loss.backward()
        opt.step()
        opt.zero_grad()
        losses.append(loss.detach())
    return losses


def train(steps: int, device: str, precision: str, batch: int = 8, seq: int = 64) -> tuple[list[float], Model, torch.Tensor]:
    """The losses of ``steps`` steps on a repeated sequence of tokens, the model, and the sequence."""
    torch.manual_seed(0)
    model = Model().to(device, torch.bfloat16 if device == "cuda" else torch.float32)
    if device == "cuda":
        opt = ab.AdamBridge(model.parameters(), lr=3e-3, precision=precision)
    else:
        opt = torch.optim.AdamW(model.parameters(), lr=3e-3)
    pattern = torch.randperm(512)[:16]   # no token twice: the tokens before say which comes next
    ids = pattern.repeat(seq // 16 + 2).to(device)
    losses = fit(model, opt, ids, steps, batch, seq)
    return [loss.item() for loss in losses], model, ids


@torch.no_grad()
def decode(model: Model, prompt: torch.Tensor, tokens: int) -> torch.Tensor:
    """``tokens`` greedy tokens after ``prompt`` [seq], one at a time."""
    ids = prompt[None]
    for _ in range(tokens):
        ids = torch.cat((ids, model.head(model(ids)[:, -1]).argmax(-1, keepdim=True)), 1)
    return ids[0, len(prompt):]


def main() -> None:
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--steps", type=int, default=60)
    parser.add_argument("--device", default="cuda" if torch.cuda.is_available() else "cpu")
    parser.add_argument("--precision", default="bf16", choices=("fp32", "bf16", "fp8"))
    args = parser.parse_args()
    losses, model, ids = train(args.steps, args.device, args.precision)
    for step in range(0, len(losses), max(1, len(losses) // 10)):
        print(f"step {step:4d}  loss {losses[step]:.4f}")
    got = decode(model, ids[:24], 16)
    print("decoded", got.tolist(), "of", ids[24:40].tolist())


if __name__ == "__main__":
    main()
