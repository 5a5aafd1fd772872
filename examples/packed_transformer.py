"""A small causal transformer on packed sequences: layer norm, packed attention and AdamW together.

    python examples/packed_transformer.py [--steps 300] [--bits 8]

Trains on documents of different lengths, each a random pattern of tokens repeated, packed one after another without
padding; the whole step (forward, backward, update) is recorded once as a HIP graph and replayed.  Then it continues
prompts token by token: one query of each request against its own keys and values.
"""
import argparse
import sys
from pathlib import Path

import numpy as np

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

import rushlite_amd as rsl  # noqa: E402
from rushlite_amd.nets import layers  # noqa: E402

VOCAB, FEATURES, HEADS, KV_HEADS, BLOCKS = 16, 64, 4, 2, 2
LENGTHS = [96, 33, 64, 17, 80, 1, 50, 43]


def linear(n_in, n_out):
    """A Linear with weights of a size that trains (the layer's own start is randn(0, 1))."""
    layer = layers.Linear(n_in, n_out)
    layer.weights = rsl.randn(0, n_in ** -0.5, [n_in, n_out], requires_grad=True)
    layer.bias = rsl.zeros([n_out], requires_grad=True)
    return layer


class Block(rsl.Module):
    def __init__(self):
        super().__init__()
        self.norm1, self.norm2 = layers.LayerNorm(FEATURES), layers.LayerNorm(FEATURES)
        self.attention = layers.SelfAttention(FEATURES, HEADS, KV_HEADS)
        self.attention.qkv = linear(FEATURES, (HEADS + 2 * KV_HEADS) * (FEATURES // HEADS))
        self.attention.out = linear(FEATURES, FEATURES)
        self.up, self.down = linear(FEATURES, 4 * FEATURES), linear(4 * FEATURES, FEATURES)

    def mlp(self, x):
        return x + self.down(self.up.forward_relu(self.norm2(x)))

    def forward(self, x, plan):
        return self.mlp(x + self.attention(self.norm1(x), plan))

    def token(self, x, cache):
        """One new token of every request; `cache` holds each request's keys and values as arrays."""
        rows = self.attention.qkv(self.norm1(x)).numpy()
        d, q_width, k_width = self.attention.head_dim, FEATURES, KV_HEADS * (FEATURES // HEADS)
        for i, row in enumerate(rows):
            for name, at in (("k", q_width), ("v", q_width + k_width)):
                cache[i][name] = np.concatenate([cache[i][name], row[None, at:at + k_width]])
        plan = self.attention.plan([1] * len(cache), [len(c["k"]) for c in cache])
        k, v = (rsl.Variable(np.concatenate([c[name] for c in cache])) for name in "kv")
        q = rsl.Variable(np.ascontiguousarray(rows[:, :q_width]))
        return self.mlp(x + self.attention.out(rsl.attention(q, k, v, plan, d ** -0.5)))


class Model(rsl.Module):
    def __init__(self, positions):
        super().__init__()
        self.tokens = rsl.randn(0, 0.5, [VOCAB, FEATURES], requires_grad=True)
        self.places = rsl.randn(0, 0.5, [positions, FEATURES], requires_grad=True)
        self.positions = positions
        for i in range(BLOCKS):
            setattr(self, f"block{i}", Block())
        self.norm, self.head = layers.LayerNorm(FEATURES), linear(FEATURES, VOCAB)
        self.softmax = layers.Softmax(dim=-1)

    def embed(self, token_rows, place_rows):
        return rsl.matmul(token_rows, self.tokens) + rsl.matmul(place_rows, self.places)

    def forward(self, token_rows, place_rows, plan):
        x = self.embed(token_rows, place_rows)
        for i in range(BLOCKS):
            x = getattr(self, f"block{i}")(x, plan)
        with rsl.capture_on():
            return self.softmax(self.head(self.norm(x)))

    def token(self, token_rows, place_rows, caches):
        x = self.embed(token_rows, place_rows)
        for i in range(BLOCKS):
            x = getattr(self, f"block{i}").token(x, caches[i])
        return self.head(self.norm(x)).numpy()


def one_hot(indices, n):
    return np.eye(n, dtype=np.float32)[indices]


def batch(rng):
    """Tokens, places and the targets of a packed batch; the first period of a document cannot be foretold."""
    tokens, places, targets = [], [], []
    for n in LENGTHS:
        period = int(rng.integers(2, 6))
        text = np.resize(rng.integers(0, VOCAB, period), n + 1)
        tokens.append(text[:n])
        places.append(np.arange(n))
        weight = (np.arange(n) + 1 >= period).astype(np.float32)
        targets.append(one_hot(text[1:], VOCAB) * weight[:, None])
    return [one_hot(np.concatenate(tokens), VOCAB), one_hot(np.concatenate(places), max(LENGTHS)),
            np.concatenate(targets)]


def train(steps, bits, seed=0, report=print):
    rng = np.random.default_rng(seed)
    rsl.manual_seed(seed)
    model = Model(max(LENGTHS))
    opt = rsl.optim.AdamW(model, lr=3e-3, weight_decay=lambda p: 0.01 if len(p.shape) > 1 else 0.0, bits=bits)
    plan = model.block0.attention.plan(LENGTHS)
    inputs = [rsl.Variable(a) for a in batch(rng)]

    def step():
        opt.zero_grad()
        probs = model(inputs[0], inputs[1], plan)
        loss = (-inputs[2] * rsl.log(probs + 1e-6)).sum(1).sum(0) * (1.0 / sum(LENGTHS))
        loss.backward()
        opt.step()
        return loss

    losses = [step().tolist()[0]]  # compiles the fused kernels
    graph = rsl.hip.Graph()
    with graph.capture():
        loss = step()
    for i in range(1, steps):
        for held, fresh in zip(inputs, batch(rng)):
            held.data.copy(rsl.Variable(fresh).data)
        graph.replay()
        losses.append(loss.tolist()[0])
        if i % 50 == 0:
            report(f"step {i}: loss {np.mean(losses[-20:]):.4f}")
    return model, losses


def continue_prompts(model, prompts, new_tokens):
    """Greedy continuations, one token of every request at a time."""
    empty = np.zeros((0, KV_HEADS * (FEATURES // HEADS)), np.float32)
    caches = [[dict(k=empty, v=empty) for _ in prompts] for _ in range(BLOCKS)]
    texts = [[] for _ in prompts]
    longest = max(len(p) for p in prompts)
    # Requests start so that their prompts end together: each joins when its first token is due.
    for t in range(longest + new_tokens):
        live = [i for i, p in enumerate(prompts) if t >= longest - len(p)]
        for i in live:
            if len(texts[i]) < len(prompts[i]):
                texts[i].append(int(prompts[i][len(texts[i])]))
        rows = [one_hot([texts[i][-1] for i in live], VOCAB), one_hot([len(texts[i]) - 1 for i in live], model.positions)]
        with rsl.no_grad():
            held = [[c[i] for i in live] for c in caches]
            logits = model.token(*(rsl.Variable(r) for r in rows), held)
        for i, row in zip(live, logits):
            if len(texts[i]) >= len(prompts[i]) and len(texts[i]) < len(prompts[i]) + new_tokens:
                texts[i].append(int(row.argmax()))
    return [x[len(p):] for x, p in zip(texts, prompts)]


if __name__ == "__main__":
    parser = argparse.ArgumentParser()
    parser.add_argument("--steps", type=int, default=300)
    parser.add_argument("--bits", type=int, default=8, choices=(8, 32))
    args = parser.parse_args()
    model, losses = train(args.steps, args.bits)
    print(f"loss {losses[0]:.3f} -> {np.mean(losses[-20:]):.3f}")
    prompts = [np.resize([3, 7, 1], 14), np.resize([5, 2], 9), np.resize([9, 4, 11, 0], 20)]
    for prompt, text in zip(prompts, continue_prompts(model, prompts, 8)):
        print(prompt.tolist(), "->", text)
