"""A small recurrent language model of this library's parts, distilled from a teacher's top logits and run token by token.

RecurrentStudent is a residual stream with, in every layer, a norm and an LSTM, a norm and attention with a decaying state, and
at the end a norm and the logits.  Both mixers carry a state of fixed size, so that a token costs the same however long the text
in front of it is.  `python -m flashlstm_poc_amd.student` trains one against a teacher that knows which tokens may follow which,
then continues a prompt token by token.

The reference has no language model; this runs layer_norm, decay_attention, decay_attention_step and distillation_train /
distillation_loss together with StackedLSTM as a user's program would.
"""
from __future__ import annotations

import argparse
from typing import List, NamedTuple, Optional, Tuple

import torch

from .lm_ops import LayerNorm, decay_attention, decay_attention_step, distillation_loss
from .stack import StackedLSTM


class LayerState(NamedTuple):
    """What a layer carries from token to token: the LSTM's h and c (1, B, width) and the attention's (B, heads, d, d)."""
    h: torch.Tensor
    c: torch.Tensor
    memory: torch.Tensor


class RecurrentLayer(torch.nn.Module):
    """Norm, LSTM, norm, attention with a decaying state; each reads the residual stream and returns what is to be added to it, which
    the next norm does."""

    def __init__(self, width: int, heads: int, device="cuda"):
        super().__init__()
        if heads < 1 or width % heads != 0:
            raise ValueError(f"width ({width}) must be a multiple of the number of heads ({heads})")
        self.heads = heads
        self.norm_lstm, self.norm_attention = LayerNorm(width, device=device), LayerNorm(width, device=device)
        self.lstm = StackedLSTM(width, width, 1, device=device)
        self.qkv = torch.nn.Linear(width, 3 * width, bias=False, device=device)
        self.out = torch.nn.Linear(width, width, bias=False, device=device)
        # memories of 2 to 2^8 tokens, longer from head to head
        reach = torch.exp2(torch.linspace(1, 8, heads, device=device))
        self.register_buffer("log_decay", torch.log1p(-1 / reach))

    def _heads(self, y):
        qkv = torch.nn.functional.linear(y, self.qkv.weight.to(y.dtype))
        return qkv.unflatten(-1, (3, self.heads, -1)).unbind(-3)

    def _join(self, o):
        return torch.nn.functional.linear(o.flatten(-2), self.out.weight.to(o.dtype))

    def forward(self, stream, added, state: Optional[LayerState]):
        """stream, added (T, B, width) fp16, added None in front of the first layer -> stream, added, LayerState."""
        y, stream = (self.norm_lstm(stream), stream) if added is None else self.norm_lstm(stream, added)
        added, (h, c) = self.lstm(y, None if state is None else (state.h, state.c))
        y, stream = self.norm_attention(stream, added)
        q, k, v = (t.transpose(0, 1) for t in self._heads(y))     # (B, T, heads, d), as they lie
        o, memory = decay_attention(q, k, v, self.log_decay, state=None if state is None else state.memory)
        return stream, self._join(o.transpose(0, 1)), LayerState(h, c, memory)

    def step(self, stream, added, state: LayerState):
        """The same for one token, stream and added (1, B, width); state.memory is updated in place."""
        y, stream = (self.norm_lstm(stream), stream) if added is None else self.norm_lstm(stream, added)
        added, (h, c) = self.lstm(y, (state.h, state.c))
        y, stream = self.norm_attention(stream, added)
        q, k, v = self._heads(y[0])
        o = decay_attention_step(q, k, v, self.log_decay, state.memory)
        return stream, self._join(o)[None], LayerState(h, c, state.memory)


class RecurrentStudent(torch.nn.Module):
    """Tokens (T, B) -> logits (T, B, vocabulary) fp16; parameters fp32, activations fp16."""

    def __init__(self, vocabulary: int, width: int, heads: int, layers: int = 1, device="cuda"):
        super().__init__()
        self.embedding = torch.nn.Embedding(vocabulary, width, device=device)
        self.layers = torch.nn.ModuleList(RecurrentLayer(width, heads, device) for _ in range(layers))
        self.norm = LayerNorm(width, device=device)
        self.head = torch.nn.Linear(width, vocabulary, bias=False, device=device)

    def _logits(self, stream, added):
        y = self.norm(stream) if added is None else self.norm(stream, added)[0]
        return torch.nn.functional.linear(y, self.head.weight.to(y.dtype))

    def forward(self, tokens, state: Optional[List[LayerState]] = None) -> Tuple:
        """A prompt or a training batch from `state` (None: the beginning) -> logits of all positions, state behind them."""
        stream, added, out = self.embedding(tokens).half(), None, []
        for i, layer in enumerate(self.layers):
            stream, added, after = layer(stream, added, None if state is None else state[i])
            out.append(after)
        return self._logits(stream, added), out

    @torch.no_grad()
    def step(self, tokens, state: List[LayerState]) -> Tuple:
        """One token of every sequence, tokens (B,) -> logits (B, vocabulary), state; the memories in `state` are updated in place."""
        stream, added, out = self.embedding(tokens)[None].half(), None, []
        for layer, before in zip(self.layers, state):
            stream, added, after = layer.step(stream, added, before)
            out.append(after)
        return self._logits(stream, added)[0], out

    @torch.no_grad()
    def generate(self, prompt, count: int):
        """The `count` likeliest tokens behind prompt (T, B), one after the other -> (count, B)."""
        out = torch.empty((count, prompt.shape[1]), device=prompt.device, dtype=torch.int64)
        logits, state = self(prompt)
        logits = logits[-1]
        for i in range(count):
            if i > 0:
                logits, state = self.step(out[i - 1], state)
            out[i] = logits.argmax(-1)
        return out


def successor_teacher(vocabulary: int, top: int, seed: int = 0, device="cuda"):
    """A teacher as a table: for each token the `top` tokens that may follow it, (vocabulary, top) int32, and their logits, fp32, the
    first well ahead of the others."""
    g = torch.Generator(device=device).manual_seed(seed)
    index = torch.stack([torch.randperm(vocabulary, device=device, generator=g)[:top] for _ in range(vocabulary)]).to(torch.int32)
    logits = torch.sort(torch.randn(vocabulary, top, device=device, generator=g), descending=True).values
    logits[:, 0] += 3
    return logits, index


def train(student: RecurrentStudent, teacher, steps: int, *, length: int = 64, batch: int = 16, temperature: float = 1.0, rate: float = 3e-3,
          seed: int = 0, loss_scale: float = 4096.0, report=None) -> List[float]:
    """Distils `teacher` (logits, index by token) into the student on random texts; returns the mean loss of every step.

    loss_scale: on the mean, so that fp16 gradients of a logit (about 1 / (rows * vocabulary)) lie in that type's range; taken out
    of the parameters' gradients."""
    logits, index = teacher
    device = logits.device
    g = torch.Generator(device=device).manual_seed(seed)
    optimizer = torch.optim.Adam(student.parameters(), lr=rate)
    losses = []
    for step in range(steps):
        tokens = torch.randint(0, logits.shape[0], (length, batch), device=device, generator=g)
        out, _ = student(tokens)
        loss = distillation_loss(out, logits[tokens], index[tokens], temperature=temperature).mean()
        optimizer.zero_grad(set_to_none=True)
        (loss * loss_scale).backward()
        for p in student.parameters():
            p.grad.div_(loss_scale)
        optimizer.step()
        losses.append(loss.detach())
        if report is not None and (step % 20 == 0 or step == steps - 1):
            report(step, float(losses[-1]))
    return [float(v) for v in losses]


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--vocabulary", type=int, default=1000)
    ap.add_argument("--width", type=int, default=256)
    ap.add_argument("--heads", type=int, default=4)
    ap.add_argument("--layers", type=int, default=1)
    ap.add_argument("--top", type=int, default=8)
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--length", type=int, default=64)
    ap.add_argument("--batch", type=int, default=32)
    a = ap.parse_args()
    torch.manual_seed(0)
    student = RecurrentStudent(a.vocabulary, a.width, a.heads, a.layers)
    teacher = successor_teacher(a.vocabulary, a.top)
    train(student, teacher, a.steps, length=a.length, batch=a.batch, report=lambda s, v: print(f"step {s:5d}  loss {v:.4f}", flush=True))
    prompt = torch.randint(0, a.vocabulary, (8, 4), device="cuda")
    out = student.generate(prompt, 16)
    follows = torch.cat([prompt[-1:], out])
    right = (teacher[1][follows[:-1].long(), 0] == follows[1:]).float().mean()
    print(f"tokens that are the teacher's first choice: {100 * float(right):.0f} %")


if __name__ == "__main__":
    main()
