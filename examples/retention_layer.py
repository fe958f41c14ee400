"""A small language model of retention layers: the matrix-state operators of this package together, as they are used.

    python examples/retention_layer.py            # a few training steps, then a prompt and single tokens

A layer norms the residual stream (``rms_norm`` with the residual's addition), projects it to queries, keys, values and decays,
turns the positions in (``rotary``), runs the recurrence over them (``linear_attention``) and projects back.  A prompt goes
through the same layers without gradients and leaves their states; every further token takes ``linear_attention_step``, which
updates the states in place.  Projections are plain matrix products; documents in one row are kept apart by an empty state.
"""
from __future__ import annotations

import argparse
import math
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from fast_sequential_scan_b200 import linear_attention, linear_attention_step, rms_norm, rotary, rotary_turns  # noqa: E402


class RetentionLayer(torch.nn.Module):
    def __init__(self, width: int, heads: int, key_heads: int, head_dim: int):
        super().__init__()
        self.heads, self.key_heads, self.head_dim = heads, key_heads, head_dim
        self.norm = torch.nn.Parameter(torch.ones(width))
        self.qkv = torch.nn.Linear(width, (2 * heads + key_heads) * head_dim, bias=False)
        self.decay = torch.nn.Linear(width, heads)
        self.out_norm = torch.nn.Parameter(torch.ones(head_dim))
        self.out = torch.nn.Linear(heads * head_dim, width, bias=False)
        with torch.no_grad():      # memories from some ten to some thousand tokens to begin with
            self.decay.bias.copy_(torch.linspace(2.0, 7.0, heads))

    def project(self, x, residual, starts=None):
        """``(residual stream, q, k, v, log_decay)`` of ``x`` ``[batch, seq, width]``."""
        y, residual = rms_norm(x, self.norm, residual=residual)
        H, Hk, D = self.heads, self.key_heads, self.head_dim
        q, k, v = self.qkv(y).split([H * D, Hk * D, H * D], dim=-1)
        log_decay = torch.nn.functional.logsigmoid(self.decay(y).float())
        if starts is not None:
            log_decay = log_decay.masked_fill(starts[..., None], -math.inf)
        return residual, q.unflatten(-1, (H, D)), k.unflatten(-1, (Hk, D)), v.unflatten(-1, (H, D)), log_decay

    def finish(self, o):
        return self.out(rms_norm(o, self.out_norm).flatten(-2))

    def forward(self, x, residual, positions, turns, *, starts=None, state=None, lengths=None, keep_state=False):
        residual, q, k, v, log_decay = self.project(x, residual, starts)
        q, k = rotary(q, k, positions, turns)
        o = linear_attention(q, k, v, log_decay, h0=state, lengths=lengths, return_final_state=keep_state)
        o, state = o if keep_state else (o, None)
        return self.finish(o), residual, state

    def step(self, x, residual, positions, turns, state, slots):
        """One token for each sequence, ``x`` ``[batch, 1, width]``; ``state`` is updated in place."""
        residual, q, k, v, log_decay = self.project(x, residual)
        q, k = rotary(q, k, positions, turns)
        o = linear_attention_step(q[:, 0], k[:, 0], v[:, 0], log_decay[:, 0], state, slots=slots)
        return self.finish(o[:, None]), residual


class RetentionModel(torch.nn.Module):
    def __init__(self, vocabulary: int = 512, width: int = 768, layers: int = 2, heads: int = 12, key_heads: int = 4, head_dim: int = 64):
        super().__init__()
        self.embed = torch.nn.Embedding(vocabulary, width)
        self.layers = torch.nn.ModuleList(RetentionLayer(width, heads, key_heads, head_dim) for _ in range(layers))
        self.norm = torch.nn.Parameter(torch.ones(width))
        turns, _ = rotary_turns(head_dim)
        self.register_buffer("turns", turns, persistent=False)

    def logits(self, x, residual):
        y, _ = rms_norm(x, self.norm, residual=residual)
        return torch.nn.functional.linear(y, self.embed.weight)

    def forward(self, tokens, *, starts=None, states=None, first=0, lengths=None, keep_states=False):
        """Logits ``[batch, seq, vocabulary]`` (and the layers' states).  ``starts``: where a document begins; ``first``: the
        position of the first token, a number or one for each sequence."""
        B, T = tokens.shape
        positions = torch.arange(T, device=tokens.device) + torch.as_tensor(first, device=tokens.device).reshape(-1, 1)
        x, residual, kept = self.embed(tokens), None, []
        residual = torch.zeros_like(x)
        for i, layer in enumerate(self.layers):
            x, residual, state = layer(x, residual, positions.expand(B, T), self.turns, starts=starts, state=states[i] if states else None,
                                       lengths=lengths, keep_state=keep_states)
            kept.append(state)
        logits = self.logits(x, residual)
        return (logits, kept) if keep_states else logits

    def step(self, tokens, positions, states, slots=None):
        """Logits ``[batch, vocabulary]`` of one further token for each sequence."""
        x = self.embed(tokens)[:, None]
        residual = torch.zeros_like(x)
        for layer, state in zip(self.layers, states):
            x, residual = layer.step(x, residual, positions[:, None], self.turns, state, slots)
        return self.logits(x, residual)[:, 0]


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=20)
    ap.add_argument("--batch", type=int, default=4)
    ap.add_argument("--seq", type=int, default=512)
    a = ap.parse_args()
    torch.manual_seed(0)
    model = RetentionModel().cuda().to(torch.bfloat16)
    optimizer = torch.optim.AdamW(model.parameters(), lr=1e-3)
    # a sequence to learn: every document counts up from a random token
    for i in range(a.steps):
        starts = torch.rand(a.batch, a.seq + 1, device="cuda") < 1 / 64
        starts[:, 0] = True
        begin = torch.randint(0, 512, starts.shape, device="cuda")
        at = torch.arange(a.seq + 1, device="cuda").expand_as(starts)
        last = torch.where(starts, at, 0).cummax(1).values
        tokens = (begin.gather(1, last) + at - last) % 512
        loss = torch.nn.functional.cross_entropy(model(tokens[:, :-1], starts=starts[:, :-1]).float().flatten(0, 1), tokens[:, 1:].flatten())
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        if i % 5 == 0 or i == a.steps - 1:
            print(f"step {i}: loss {loss.item():.3f}")
    with torch.no_grad():
        lengths = torch.tensor([40, 17, 1, 33], device="cuda", dtype=torch.int32)
        prompt = (torch.arange(40, device="cuda") + 100 * torch.arange(4, device="cuda")[:, None]) % 512
        logits, states = model(prompt, lengths=lengths, keep_states=True)
        token = logits[torch.arange(4, device="cuda"), lengths.long() - 1].argmax(-1)
        out, positions = [token], lengths.long()
        for _ in range(8):
            token = model.step(token, positions, states).argmax(-1)
            positions = positions + 1
            out.append(token)
    print("continuations:", torch.stack(out, 1).tolist())


if __name__ == "__main__":
    main()
