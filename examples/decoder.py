"""A small decoder: rotary attention, dropout added to the residual stream, gated feed-forward blocks and a loss over the
vocabulary that never holds the logits.

    python examples/decoder.py [--steps 300] [--vocabulary 512] [--gate silu]

Trains on packed documents of different lengths, each a random pattern of tokens repeated; a document's first period is
not counted.  The whole step (forward, backward, update) is recorded once as a HIP graph and replayed: every replay drops
afresh.  Then it scores fresh documents, longer than those it was trained on.
"""
import argparse
import sys
from pathlib import Path

import numpy as np

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

import rushlite_amd as rsl  # noqa: E402
from rushlite_amd.nets import layers  # noqa: E402

FEATURES, HEADS, KV_HEADS, HIDDEN, BLOCKS, RATE = 64, 4, 2, 160, 2, 0.1
LENGTHS = [96, 33, 64, 17, 80, 1, 50, 43]


def scaled(layer):
    """A layer with weights of a size that trains (its own start is randn(0, 1)) and a bias of zeros."""
    n_in, n_out = layer.weights.shape
    layer.weights = rsl.randn(0, n_in ** -0.5, [n_in, n_out], requires_grad=True)
    layer.bias = rsl.zeros([n_out], requires_grad=True)
    return layer


class Block(rsl.Module):
    def __init__(self, generator, gate):
        super().__init__()
        self.norm1, self.norm2 = layers.LayerNorm(FEATURES), layers.LayerNorm(FEATURES)
        self.attention = layers.SelfAttention(FEATURES, HEADS, KV_HEADS, rotary=layers.Rotary(FEATURES // HEADS))
        self.mlp = layers.GatedFeedForward(FEATURES, HIDDEN, gate)
        for part in (self.attention.qkv, self.attention.out, self.mlp.up, self.mlp.down):
            scaled(part)
        self.drop = layers.RandomDropout(RATE, generator)

    def forward(self, x, plan, positions):
        x = self.drop(self.attention(self.norm1(x), plan, positions), x)
        return self.drop(self.mlp(self.norm2(x)), x)


class Decoder(rsl.Module):
    def __init__(self, vocabulary, gate="silu", seed=0):
        super().__init__()
        self.vocabulary, self.generator = vocabulary, rsl.Generator(seed)
        self.tokens = rsl.randn(0, 0.5, [vocabulary, FEATURES], requires_grad=True)
        self.blocks = [Block(self.generator, gate) for _ in range(BLOCKS)]
        for i, block in enumerate(self.blocks):
            setattr(self, f"block{i}", block)
        self.norm, self.loss = layers.LayerNorm(FEATURES), layers.VocabularyLoss(FEATURES, vocabulary)
        scaled(self.loss.head)

    def train(self, active):
        for block in self.blocks:
            block.drop.active = active

    def features(self, token_rows, plan, positions):
        x = rsl.matmul(token_rows, self.tokens)
        for block in self.blocks:
            x = block(x, plan, positions)
        return self.norm(x)

    def forward(self, token_rows, targets, plan, positions):
        return self.loss(self.features(token_rows, plan, positions), targets)


def batch(rng, vocabulary, lengths):
    """The tokens of a packed batch as one-hot rows, and the targets, negative in each document's first period."""
    tokens, targets = [], []
    for n in lengths:
        period = int(rng.integers(2, 6))
        text = np.resize(rng.integers(0, vocabulary, period), n + 1)
        tokens.append(text[:n])
        targets.append(np.where(np.arange(n) + 1 >= period, text[1:], -1))
    return np.eye(vocabulary, dtype=np.float32)[np.concatenate(tokens)], np.concatenate(targets).astype(np.int64)


def variables(rows, targets):
    return rsl.Variable(rows), rsl.Variable(targets, dtype=rsl.dtype.int64)


def train(steps, vocabulary=512, gate="silu", seed=0, report=print):
    rng = np.random.default_rng(seed)
    rsl.manual_seed(seed)
    model = Decoder(vocabulary, gate, seed)
    opt = rsl.optim.AdamW(model, lr=3e-3, weight_decay=lambda p: 0.01 if len(p.shape) > 1 else 0.0)
    plan, positions = model.block0.attention.plan(LENGTHS), layers.packed_positions(LENGTHS)
    inputs = variables(*batch(rng, vocabulary, LENGTHS))

    def step():
        opt.zero_grad()
        loss = model(*inputs, plan, positions)
        loss.backward()
        opt.step()
        return loss

    losses = [step().tolist()[0]]
    graph = rsl.hip.Graph()
    with graph.capture():
        loss = step()
    for i in range(1, steps):
        for held, fresh in zip(inputs, variables(*batch(rng, vocabulary, LENGTHS))):
            held.data.copy(fresh.data)
        graph.replay()
        losses.append(loss.tolist()[0])
        if i % 50 == 0:
            report(f"step {i}: loss {np.mean(losses[-20:]):.4f}")
    return model, losses


def score(model, lengths, seed=1):
    """Each document's mean loss on what can be foretold of it."""
    rows, targets = batch(np.random.default_rng(seed), model.vocabulary, lengths)
    model.train(False)
    with rsl.no_grad():
        x, t = variables(rows, targets)
        each = model.loss.rows(model.features(x, model.block0.attention.plan(lengths), layers.packed_positions(lengths)), t)
    model.train(True)
    ends = np.cumsum(lengths)
    return [float(each.numpy()[e - n:e][targets[e - n:e] >= 0].mean()) for n, e in zip(lengths, ends)]


if __name__ == "__main__":
    parser = argparse.ArgumentParser()
    parser.add_argument("--steps", type=int, default=300)
    parser.add_argument("--vocabulary", type=int, default=512)
    parser.add_argument("--gate", default="silu", choices=("silu", "gelu", "gelu_tanh", "relu", "sigmoid"))
    args = parser.parse_args()
    model, losses = train(args.steps, args.vocabulary, args.gate)
    print(f"loss {losses[0]:.3f} -> {np.mean(losses[-20:]):.3f}; {model.generator.calls} calls of the generator")
    print("fresh documents of 40, 90 and 140 tokens:", [round(v, 3) for v in score(model, [40, 90, 140])])
