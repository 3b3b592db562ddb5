"""Distil a token model into a smaller one on the xdna device, then let the student write.

    python examples/distill_student.py [--steps N]

Both models predict the next token from the current one: embed -> gated feed-forward block with
a residual -> head.  The teacher is fixed (random weights; there is no data to download).  Per
step it names its most likely next tokens for a batch (``token_log_probs``), and the student is
trained on them (``distill_loss``).  Afterwards the student continues a few prompts one token at
a time, and the teacher scores what it wrote.
"""
import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "pytorch-xdna2_amd"))

import xdna_train  # noqa: E402,F401  (registers the device)
from xdna_train import tokens  # noqa: E402

VOCAB, TOP = 1000, 32


class NextToken(torch.nn.Module):
    def __init__(self, width: int, hidden: int, seed: int, head_scale: float):
        super().__init__()
        g = torch.Generator().manual_seed(seed)

        def normal(*shape, std):
            return torch.nn.Parameter((torch.randn(*shape, generator=g) * std).bfloat16())

        self.table = normal(VOCAB, width, std=width**-0.5)
        self.w_in = normal(2 * hidden, width, std=width**-0.5)
        self.w_out = normal(width, hidden, std=hidden**-0.5)
        self.head = normal(width, VOCAB, std=head_scale * width**-0.5)

    def forward(self, ids):
        x = tokens.embed(ids, self.table, scale=self.table.shape[1] ** 0.5)
        h = x + tokens.gated_mlp(x, self.w_in, self.w_out, "silu")
        return (h.reshape(-1, h.shape[-1]) @ self.head).view(*ids.shape, VOCAB)


def main(steps: int = 300, batch: int = 8, length: int = 128, report: int = 50) -> dict:
    dev = torch.device("xdna")
    teacher = NextToken(256, 640, seed=1, head_scale=2.0).to(dev).requires_grad_(False)
    student = NextToken(128, 320, seed=2, head_scale=0.5).to(dev)
    opt = torch.optim.Adam(student.parameters(), lr=3e-3, fused=True)
    g = torch.Generator().manual_seed(3)
    unscored = torch.full((batch, length), -1, device=dev)
    losses = []
    for step in range(steps):
        ids = torch.randint(0, VOCAB, (batch, length), generator=g).to(dev)
        top = tokens.token_log_probs(teacher(ids), unscored, top_k=TOP)
        loss = tokens.distill_loss(student(ids), top.top_ids, top.top_log_probs)
        opt.zero_grad(set_to_none=True)
        loss.backward()
        opt.step()
        if step % report == 0 or step == steps - 1:
            losses.append(float(loss.detach()))
            print(f"step {step:4d}  loss {losses[-1]:.4f}", flush=True)

    prompts = torch.arange(4, device=dev)
    with torch.no_grad():
        now, text = prompts, []
        for _ in range(16):  # one token of every text per step
            now = tokens.token_log_probs(student(now), torch.full_like(now, -1), top_k=1).top_ids[:, 0]
            text.append(now)
        text = torch.stack(text, dim=1)
        before = torch.cat([prompts[:, None], text[:, :-1]], dim=1)
        by_teacher = tokens.token_log_probs(teacher(before), text)
        by_chance = tokens.token_log_probs(teacher(before), (text + VOCAB // 2) % VOCAB)
    written = float(by_teacher.log_probs.mean())
    chance = float(by_chance.log_probs.mean())
    print(f"teacher's mean log probability of the student's tokens {written:.3f}, of others {chance:.3f}; "
          f"its entropy there {float(by_teacher.entropy.mean()):.3f}")
    return {"losses": losses, "written": written, "chance": chance, "text": text.cpu()}


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--steps", type=int, default=300)
    main(parser.parse_args().steps)
