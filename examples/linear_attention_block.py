"""One block of a language model with linear attention, as a server runs it: prompts first, then a token at a time.

    python examples/linear_attention_block.py [--batch 4] [--tokens 500] [--steps 8] [--width 512] [--heads 8] [--dtype f32|bf16]

    x ---------------------------------------------------------------(+)--> s, and norm(s) for the block behind
    norm -> connected: q, k, v, gate, decay -> linear attention ->     |
            norm of each head * silu(gate) -> connected -> norm * scale

The projections are connected layers, the rest the operators of linear attention and of the norms around it.  The script
runs the prompts, then `steps` tokens on the states they left, and checks that prompts that hold those tokens too give the same.
"""
import argparse
import sys
from pathlib import Path

if str(Path(__file__).resolve().parent.parent) not in sys.path:
    sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

import torch

from nebula_b200 import api


class Block:
    def __init__(self, handle, width, heads, head_dim, dtype="f32", seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        rand = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
        self.handle, self.width, self.heads, self.dim, self.dtype = handle, width, heads, head_dim, dtype
        self.inner = heads * head_dim
        self.outs = 4 * self.inner + heads              # q, k, v, gate, and a decay for each head
        self.w_in, self.w_out = rand(self.outs, width) / width ** 0.5, rand(width, self.inner) / self.inner ** 0.5
        self.norm_in, self.norm_heads, self.norm_out, self.norm_next = (1 + 0.1 * rand(n) for n in (width, self.inner, width, width))
        self.scale = 0.5 + 0.1 * rand(width)
        self.plans = {}

    def plan(self, key, make):
        if key not in self.plans:
            self.plans[key] = make()
            self.plans[key].prepare()
        return self.plans[key]

    def connected(self, x, name):
        weight = getattr(self, "w_" + name)

        def make():
            layer = api.Connected(self.handle, x.shape[0], weight.shape[1], weight.shape[0], activation="linear")
            layer.set_weights(weight, torch.zeros(weight.shape[0], device="cuda"))
            return layer
        return self.plan(("connected", x.shape[0], name), make).forward(x)

    def forward(self, x, state, single):
        """x [batch, tokens, width], or [batch, width] for a token of each; `state` is updated."""
        lead, kind = x.shape[:-1], torch.float32 if self.dtype == "f32" else torch.bfloat16
        h, _ = self.handle.norm_gate_residual(x, self.norm_in)
        y = self.connected(h.reshape(-1, self.width), "in").view(*lead, self.outs)
        q, k, v, gate = (y[..., i * self.inner:(i + 1) * self.inner].to(kind).view(*lead, self.heads, self.dim) for i in range(4))
        k = k / self.dim ** 0.5
        decay = torch.nn.functional.logsigmoid(y[..., 4 * self.inner:] + 3)
        layer = self.plan(("attention", *lead), lambda: api.LinearAttention(self.handle, lead[0], 1 if single else lead[1], self.heads, self.dim,
                                                                              self.dim, dtype=self.dtype, scale=self.dim ** -0.5))
        o = layer.step(q, k, v, decay, state) if single else layer.forward(q, k, v, decay, state=state, state_out=state)
        o, _ = self.handle.norm_gate_residual(o.view(-1, self.inner), self.norm_heads, groups=self.heads, gate=gate.reshape(-1, self.inner))
        o = self.connected(o.float(), "out").view(*lead, self.width)
        return self.handle.norm_gate_residual(o, self.norm_out, residual=x, channel_scale=self.scale, next_norm="rms", next_weight=self.norm_next)

    def state(self, batch):
        return torch.zeros(batch, self.heads, self.dim, self.dim, device="cuda")

    def close(self):
        for p in self.plans.values():
            p.close()


def run(handle, batch=4, tokens=500, steps=8, width=512, heads=8, head_dim=64, dtype="f32"):
    """Largest relative differences (2-norms) of the stepped tokens' outputs and of the states, against prompts that hold them."""
    block = Block(handle, width, heads, head_dim, dtype)
    x = torch.randn(batch, tokens + steps, width, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    whole = block.state(batch)
    s_all, y_all = block.forward(x, whole, False)
    state = block.state(batch)
    block.forward(x[:, :tokens].contiguous(), state, False)
    off = 0.0
    for t in range(tokens, tokens + steps):
        s, y = block.forward(x[:, t].contiguous(), state, True)
        off = max(off, float((s - s_all[:, t]).norm() / s_all[:, t].norm()), float((y - y_all[:, t]).norm() / y_all[:, t].norm()))
    handle.synchronize()
    block.close()
    return off, float((state - whole).norm() / whole.norm())


def main():
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("batch", 4), ("tokens", 500), ("steps", 8), ("width", 512), ("heads", 8), ("head-dim", 64)):
        p.add_argument("--" + name, type=int, default=value)
    p.add_argument("--dtype", choices=("f32", "bf16"), default="f32")
    a = p.parse_args()
    handle = api.Handle(0, "tf32x3")
    out, state = run(handle, a.batch, a.tokens, a.steps, a.width, a.heads, a.head_dim, a.dtype)
    print(f"{a.steps} tokens in steps against the same in a prompt: outputs differ by {out:.1e}, states by {state:.1e}")
    handle.close()


if __name__ == "__main__":
    main()
