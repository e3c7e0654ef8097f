"""An autoregressive decoder that writes tokens from a text encoder's states.

Runs the token decoder's operators together as a program would: a prompt in one
call, then token by token, several utterances at once over one paged cache of
8-bit keys and values.  The weights are random: it shows the calls and what a
step costs, and writes no speech.

usage: python examples/decode_tokens.py [--batch 4] [--prompt 52] [--tokens 64] [--layers 4]
"""
import argparse
import importlib
import os
import sys
import time

import numpy as np

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
kk = importlib.import_module("best-tts-godot_amd")
ops = kk.ops


class Decoder:
    """Layers of self-attention over a cache, attention over text states and a
    feed-forward part, `heads` heads of 64, a vocabulary of audio codes."""

    END = 0

    def __init__(self, seed, layers=4, heads=12, vocabulary=1025):
        r = np.random.default_rng(seed)
        self.heads, self.dim, self.width, self.vocabulary = heads, 64, heads * 64, vocabulary

        def weight(rows, columns):
            w = kk.to_device((r.normal(size=(rows, columns)) / rows ** 0.5).astype(np.float16))
            return w, ops.gemm_pack(w)

        def ones(n):
            return kk.to_device(np.ones(n, np.float32))
        w = self.width
        self.embedding = kk.to_device(r.normal(size=(vocabulary, w)).astype(np.float32))
        self.layers = [dict(qkv=weight(w, 3 * w), out=weight(w, w), q=weight(w, w), kv=weight(w, 2 * w), back=weight(w, w),
                            up=weight(w, 4 * w), down=weight(4 * w, w), norms=[ones(w) for _ in range(3)], qn=ones(64),
                            kn=ones(64)) for _ in range(layers)]
        self.head, self.norm = weight(w, vocabulary), ones(w)
        self.turns = kk.to_device(kk.rotary_turns(64))

    @staticmethod
    def product(x, w):
        return ops.matmul(x, w[0], packed=w[1])

    def text(self, states):
        """Keys and values of text states [B, S, width] for each layer."""
        kv = [self.product(states, w["kv"]) for w in self.layers]
        kv = [x.reshape(x.shape[:2] + (2 * self.heads, self.dim)) for x in kv]
        return [(x.slice_axis(2, 0, self.heads), x.slice_axis(2, self.heads, 2 * self.heads)) for x in kv]

    def __call__(self, ids, starts, lengths, caches, table, text, text_lengths):
        """Logits [B, vocabulary] after tokens ids [B, T], which come at places
        starts [B] and make the sequences `lengths` [B] long."""
        B, T = ids.shape
        positions = ops.binary("Add", starts.expand_dims(1), kk.to_device(np.arange(T, dtype=np.int32)[None]))
        x = ops.gather(self.embedding, ids)
        for w, cache, (text_k, text_v) in zip(self.layers, caches, text):
            qkv = self.product(ops.layernorm(x, w["norms"][0]), w["qkv"]).reshape((B, T, 3 * self.heads, self.dim))
            q, k, v = (qkv.slice_axis(2, i * self.heads, (i + 1) * self.heads) for i in range(3))
            q, k = ops.qk_norm_rotary(q, k, positions, self.turns, w["qn"], w["kn"])
            ops.cache_append(cache, k, v, table, starts)
            y = ops.cache_attention(q, cache, table, lengths)
            x = ops.binary("Add", x, self.product(y.reshape((B, T, self.width)), w["out"]))
            q = self.product(ops.layernorm(x, w["norms"][1]), w["q"]).reshape((B, T, self.heads, self.dim))
            y = ops.cross_attention(q, text_k, text_v, text_lengths)
            x = ops.binary("Add", x, self.product(y.reshape((B, T, self.width)), w["back"]))
            y = ops.fast_gelu(self.product(ops.layernorm(x, w["norms"][2]), w["up"]))
            x = ops.binary("Add", x, self.product(y, w["down"]))
        last = x.slice_axis(1, T - 1, T).contiguous().reshape((B, self.width))
        return self.product(ops.layernorm(last, self.norm), self.head)


def generate(model, states, text_lengths, prompt, tokens, block=64):
    """Writes `tokens` tokens behind prompt [B, P] for text states [B, S, width];
    returns them [B, tokens] and the seconds that each step took."""
    B, P = prompt.shape
    columns = -(-(P + tokens) // block)
    table = kk.to_device(np.arange(B * columns, dtype=np.int32).reshape(B, columns))
    caches = [kk.KVCache.zeros(B * columns, model.heads, model.dim, block) for _ in model.layers]
    text, text_lengths = model.text(kk.to_device(states)), kk.to_device(text_lengths)
    going_on = np.ones(model.vocabulary, bool)
    going_on[model.END] = False  # an utterance does not end before its last step
    allowed = kk.to_device(kk.allowed_bits(going_on))
    repetition, frequency = (kk.to_device(np.array([x], np.float32)) for x in (1.1, 0.05))
    history, ids, seconds = prompt.astype(np.int32), prompt.astype(np.int32), []
    for i in range(tokens):
        begin = time.perf_counter()
        starts = np.full(B, 0 if i == 0 else P + i - 1, np.int32)
        logits = model(kk.to_device(ids), kk.to_device(starts), kk.to_device(starts + ids.shape[1]), caches, table, text,
                       text_lengths)
        logits = ops.process_logits(logits, kk.to_device(history), None, repetition, None, frequency, None,
                                    None if i == tokens - 1 else allowed)
        ids = kk.to_host(logits).argmax(-1).astype(np.int32)[:, None]
        history = np.concatenate([history, ids], 1)
        seconds.append(time.perf_counter() - begin)
    return history[:, P:], seconds


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("--batch", 4), ("--prompt", 52), ("--tokens", 64), ("--layers", 4)):
        ap.add_argument(name, type=int, default=value)
    a = ap.parse_args()
    kk.init()
    model = Decoder(0, a.layers)
    r = np.random.default_rng(1)
    states = r.normal(size=(a.batch, 130, model.width)).astype(np.float32)
    lengths = r.integers(65, 131, a.batch).astype(np.int32)
    prompt = r.integers(1, model.vocabulary, (a.batch, a.prompt))
    out, seconds = generate(model, states, lengths, prompt, a.tokens)
    print("tokens of the first utterance:", *out[0])
    print(f"prompt of {a.prompt} tokens: {1e3 * seconds[0]:.2f} ms, a step of {a.batch} utterances: "
          f"{1e3 * float(np.median(seconds[1:] or seconds)):.2f} ms")


if __name__ == "__main__":
    main()
