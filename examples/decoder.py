"""A small decoder trained to continue sequences, and then run token by token.

The block is a transformer's: norms of the rows, the joint projection of queries, keys and values, norms of heads and rotation
(jt.nn.qkv_norm_rope), causal attention with grouped heads from matrix products and a softmax, dropout with the residual
(jt.nn.dropout), a gated feed-forward layer (jt.nn.gated_ffn).  The task: a sequence walks through the tokens by a fixed
permutation, so that the next token follows from the last one.

    python examples/decoder.py --steps 80 --dtype float32
"""
import argparse
import os
import sys

import numpy as np

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))

import jittor_amd as jt                                     # noqa: E402
from jittor_amd import nn                                   # noqa: E402


class Decoder:
    def __init__(self, vocab=32, width=64, heads=4, kv_heads=2, dim=16, hidden=128, layers=2, longest=256, p=0.1, dtype="float32", seed=0):
        rng = np.random.default_rng(seed)
        self.vocab, self.heads, self.kv_heads, self.dim, self.p, self.dtype, self.layers = vocab, heads, kv_heads, dim, p, dtype, layers

        def weight(*shape, scale):
            return jt.array((rng.standard_normal(shape) * scale).astype(np.float32), dtype)

        self.table = nn.rope_table(longest, dim)
        self.params = {"embed": weight(vocab, width, scale=1.0), "out": weight(vocab, width, scale=width ** -0.5), "norm": jt.ones([width], dtype)}
        for i in range(layers):
            self.params.update({"%d.%s" % (i, k): v for k, v in {
                "norm1": jt.ones([width], dtype), "norm2": jt.ones([width], dtype), "q": jt.ones([dim], dtype), "k": jt.ones([dim], dtype),
                "qkv": weight((heads + 2 * kv_heads) * dim, width, scale=width ** -0.5), "proj": weight(width, heads * dim, scale=(heads * dim) ** -0.5),
                "in": weight(2 * hidden, width, scale=width ** -0.5), "down": weight(width, hidden, scale=hidden ** -0.5)}.items()})

    def _norm(self, x, scale):
        return x / ((x * x).mean([x.ndim - 1], keepdims=True) + 1e-6).sqrt() * scale

    def _attention(self, q, k, v, past):
        """q [b, heads, s, dim], k and v [b, kv_heads, past + s, dim]: token i sees the first past + i + 1."""
        b, h, s, d = q.shape
        n, group = k.shape[2], self.heads // self.kv_heads
        k, v = (u.reindex([b, h, n, d], ["i0", "i1/%d" % group, "i2", "i3"]) for u in (k, v))       # a head of keys for each of its group
        scores = nn.matmul(q, jt.transpose(k, [0, 1, 3, 2])) * float(d ** -0.5)
        seen = jt.index([s, n], 1) <= jt.index([s, n], 0) + past
        scores = jt.ternary(jt.broadcast(seen, scores.shape, [0, 1]), scores, jt.broadcast(jt.array(-1e4, self.dtype), scores.shape))
        e = (scores - scores.max([3], keepdims=True)).exp()
        return nn.matmul((e / e.sum([3], keepdims=True)).cast(self.dtype), v)      # (exp computes in float32)

    def forward(self, tokens, cache=None, train=False, step=0):
        """Logits [b, s, vocab] for tokens [b, s] (an int32 array).  `cache`: a list of one (k, v) for each layer, or Nones, which the tokens
        are appended to."""
        with jt.flag_scope(amp_reg=jt.flags.amp_reg | 36):  # sums of 16-bit values keep their type
            return self._forward(tokens, cache, train, step)

    def _forward(self, tokens, cache, train, step):
        w, (b, s) = self.params, tokens.shape
        past = 0 if cache is None or cache[0] is None else cache[0][0].shape[2]
        positions = jt.array(np.arange(past, past + s, dtype=np.int32))
        width = w["embed"].shape[1]
        x = w["embed"].reindex([b, s, width], ["@e0(i0,i1)", "i2"], extras=[jt.array(tokens.astype(np.int32))])
        for i in range(self.layers):
            p = lambda name: w["%d.%s" % (i, name)]
            qkv = nn.linear(self._norm(x, p("norm1")), p("qkv")).reshape([b, s, self.heads + 2 * self.kv_heads, self.dim])
            q, k, v = nn.qkv_norm_rope(qkv, self.heads, self.kv_heads, p("q"), p("k"), self.table, positions, heads_first=True)
            if cache is not None:
                if cache[i] is not None:
                    k, v = jt.concat([cache[i][0], k], 2), jt.concat([cache[i][1], v], 2)
                cache[i] = (k, v)
            a = jt.transpose(self._attention(q, k, v, past), [0, 2, 1, 3]).reshape([b, s, self.heads * self.dim])
            # the key of a dropout: the step; the calls of a step are told apart by their number
            x = nn.dropout(nn.linear(a, p("proj")), self.p, train, seed=step, offset=2 * i, residual=x)
            x = nn.dropout(nn.gated_ffn(self._norm(x, p("norm2")), p("in"), p("down")), self.p, train, seed=step, offset=2 * i + 1, residual=x)
        return nn.linear(self._norm(x, w["norm"]), w["out"])

    def step(self, tokens, targets, rate, step):
        """One step of gradient descent; the loss before it."""
        logits = self.forward(tokens, train=True, step=step).cast("float32")
        onehot = jt.array(np.eye(self.vocab, dtype=np.float32)[targets])
        shifted = logits - logits.max([2], keepdims=True)
        loss = ((shifted.exp().sum([2], keepdims=True).log() - shifted) * onehot).sum() / float(targets.size)
        names = list(self.params)
        grads = jt.grad(loss, [self.params[k] for k in names])
        new = [self.params[k] - g * rate for k, g in zip(names, grads)]
        jt.sync([loss] + new)
        for k, v in zip(names, new):
            self.params[k] = v.stop_grad()
        return loss.item()

    def generate(self, tokens, n):
        """The n most likely tokens behind each row, one at a time over kept keys and values."""
        cache = [None] * self.layers
        out = tokens
        for _ in range(n):
            with jt.no_grad():
                logits = self.forward(tokens, cache)
                jt.sync([logits] + [u for pair in cache for u in pair])
            tokens = logits.cast("float32").numpy()[:, -1].argmax(-1).astype(np.int32)[:, None]
            out = np.concatenate([out, tokens], 1)
        return out


def train(steps=80, batch=16, length=24, rate=0.3, dtype="float32", seed=0, report=lambda step, loss: None, **sizes):
    """(model, losses, the permutation)"""
    model = Decoder(dtype=dtype, seed=seed, **sizes)
    rng = np.random.default_rng(seed + 1)
    follows = rng.permutation(model.vocab)
    losses = []
    for step in range(steps):
        seq = [rng.integers(0, model.vocab, batch)]
        for _ in range(length):
            seq.append(follows[seq[-1]])
        seq = np.stack(seq, 1)
        losses.append(model.step(seq[:, :-1], seq[:, 1:], rate, step))
        report(step, losses[-1])
    return model, losses, follows


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=80)
    ap.add_argument("--dtype", default="float32", choices=("float32", "bfloat16", "float16"))
    a = ap.parse_args()
    model, losses, follows = train(a.steps, dtype=a.dtype, report=lambda step, loss: step % 10 or print("step %3d  loss %.4f" % (step, loss), flush=True))
    print("loss %.4f -> %.4f" % (losses[0], losses[-1]))
    start = np.arange(4, dtype=np.int32)[:, None]
    out = model.generate(start, 12)
    right = sum(int(follows[a] == b) for row in out for a, b in zip(row, row[1:]))
    print("%d of %d generated tokens follow the rule" % (right, out.size - len(out)))


if __name__ == "__main__":
    main()
