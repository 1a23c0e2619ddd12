#!/usr/bin/env python3
"""Speculative decoding of several sequences that share a prompt, over quantised K/V caches.

A decoder of the benchmark model's shape (random weights; --small for a toy one) reads a prompt
into a cache of one slot, once for all sequences, 16 rows at a time.  Then each verify pass takes a
block of every sequence (its last token and the drafts), and

  * norms the heads of the block's queries and keys, cut from the fused q|k|v output, and turns
    them to their positions (Context.qk_norm_rope),
  * quantises the block's K and V rows into the sequences' own caches as it writes them
    (Context.cache_append),
  * attends over the prompt, the sequence's own tokens and the block (Context.cache_attention),
  * scores the drafts and takes the model's own tokens with their log probabilities
    (Context.token_logprobs), or, at a temperature, keeps drafts by their probabilities and draws
    the token behind them (Context.sample_accept),

with the quantised projections in between.  Drafts that agree with the model are kept; what was
appended of the others is written over by the next block.  The drafts here are the model's own
tokens with some replaced, as no draft model is loaded.

    python3 dflash-swift_amd/examples/verify_block.py --small [--temperature 0.8]
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
import dflash_qmm  # noqa: E402

BLOCK_ROWS = 16    # most rows of a block of cache_attention


def random_linear(ctx, rows, columns, gen, bits=4, group=64):
    """A quantised layer of random codes whose values have mean 0 and variance 1 / columns."""
    words = torch.randint(-1 << 31, (1 << 31) - 1, (rows, columns * bits // 32),
                          dtype=torch.int32, device="cuda", generator=gen)
    top = (1 << bits) - 1
    scale = (12.0 / columns) ** 0.5 / (top + 1)
    scales = torch.full((rows, columns // group), scale, dtype=torch.bfloat16, device="cuda")
    biases = scales * (-top / 2)
    stock = dflash_qmm.QuantizedLinear(ctx, words, scales, biases, group_size=group, bits=bits)
    return dflash_qmm.SmallMQuantizedLinear(stock)


def norm(x):
    f = x.float()
    return (f * torch.rsqrt(f.square().mean(-1, keepdim=True) + 1e-6)).to(x.dtype)


class Decoder:
    """A decoder of `layers` blocks with quantised weights and K/V caches: `prompt` holds the
    shared tokens (one slot), `own` each sequence's."""

    def __init__(self, ctx, layers, hidden, q_heads, kv_heads, head_dim, mlp, vocab, sequences,
                 prompt_capacity, own_capacity, seed=0):
        gen = torch.Generator(device="cuda")
        gen.manual_seed(seed)
        self.ctx, self.head_dim = ctx, head_dim
        self.q_width, self.kv_width = q_heads * head_dim, kv_heads * head_dim
        self.layers = [{
            "qkv": random_linear(ctx, self.q_width + 2 * self.kv_width, hidden, gen),
            "o": random_linear(ctx, hidden, self.q_width, gen),
            "gate_up": random_linear(ctx, 2 * mlp, hidden, gen),
            "down": random_linear(ctx, hidden, mlp, gen),
            "q_norm": torch.ones(head_dim, dtype=torch.bfloat16, device="cuda"),
            "k_norm": torch.ones(head_dim, dtype=torch.bfloat16, device="cuda"),
            "prompt": dflash_qmm.KVCache(1, kv_heads, prompt_capacity, head_dim),
            "own": dflash_qmm.KVCache(sequences, kv_heads, own_capacity, head_dim),
        } for _ in range(layers)]
        self.embedding = torch.randn(vocab, hidden, device="cuda",
                                     generator=gen).to(torch.bfloat16)
        self.lm_head = random_linear(ctx, vocab, hidden, gen)
        self.rope = dflash_qmm.Rope(head_dim, base=1e6)
        self.prompt_length = 0

    def forward(self, tokens, cache, starts, lengths, prompt_length, max_length):
        """Logits [batch, rows, vocab] of blocks tokens [batch, rows] whose rows go to `cache`
        ("prompt" or "own") at starts [batch]; lengths = starts + rows."""
        ctx = self.ctx
        batch, rows = tokens.shape
        offset = prompt_length if cache == "own" else 0
        x = self.embedding[tokens.long()]
        for layer in self.layers:
            fused = layer["qkv"](norm(x))
            q, k, v = fused.split((self.q_width, self.kv_width, self.kv_width), -1)
            # v stays a slice of the fused rows; the rotated k goes back beside it
            q, heads = (t.unflatten(-1, (-1, self.head_dim)) for t in (q, k))
            q, _ = ctx.qk_norm_rope(self.rope, q, heads, layer["q_norm"], layer["k_norm"],
                                    start=offset, starts=starts, k_out=heads)
            ctx.cache_append(layer[cache], k, v, starts=starts)
            y, _ = ctx.cache_attention(
                q.flatten(2), layer[cache], lengths=lengths, max_length=max_length,
                prefix=layer["prompt"] if offset else None, prefix_length=offset or None)
            x = x + layer["o"](y)
            gate_up = layer["gate_up"](norm(x)).flatten(0, 1)
            x = x + layer["down"](ctx.silu_mul(gate_up).view(batch, rows, -1))
        return self.lm_head(norm(x))

    def read_prompt(self, tokens):
        """The shared prompt tokens [n] into the prompt caches; the last token's logits."""
        for at in range(0, tokens.shape[0], BLOCK_ROWS):
            block = tokens[None, at:at + BLOCK_ROWS]
            start = torch.full((1,), at, dtype=torch.int32, device="cuda")
            end = at + block.shape[1]
            logits = self.forward(block, "prompt", start, start + block.shape[1], 0, end)
        self.prompt_length = tokens.shape[0]
        return logits[0, -1:]

    def sample(self, blocks, starts, uniforms, temperature):
        """One pass over blocks as in verify, whose drafts are kept by their probabilities at a
        temperature: (tokens [batch, rows] -- the drafts kept and the token drawn behind them --,
        how many were kept, the chance of each, the logits).  uniforms [batch, rows] are the
        random numbers."""
        rows = blocks.shape[1]
        logits = self.forward(blocks, "own", starts, starts + rows, self.prompt_length,
                              self.layers[0]["own"].capacity)
        drafts = blocks[:, 1:].contiguous() if rows > 1 else None
        return *self.ctx.sample_accept(logits, uniforms, drafts, temperature=temperature), logits

    def verify(self, blocks, starts, top_k=5):
        """One pass over blocks [batch, rows] (a sequence's last token, then its drafts) placed
        at starts [batch] of the sequences' own tokens.  Returns per sequence how many drafts
        agree with the model, the model's tokens [batch, rows], their log probabilities, those
        of the drafts, and each row's entropy and alternatives."""
        batch, rows = blocks.shape
        own = self.layers[0]["own"]
        logits = self.forward(blocks, "own", starts, starts + rows, self.prompt_length,
                              own.capacity)
        drafts = torch.full_like(blocks, -1)      # a block's last row has none
        drafts[:, :-1] = blocks[:, 1:]
        scores, entropy, top, top_scores = self.ctx.token_logprobs(
            logits.flatten(0, 1), drafts.flatten(), top_k=top_k)
        taken = top[:, 0].view(batch, rows)
        agree = (taken == drafts)[:, :-1].int().cumprod(-1).sum(-1).int()
        return {"accepted": agree, "tokens": taken,
                "token_logprobs": top_scores[:, 0].view(batch, rows),
                "draft_logprobs": scores.view(batch, rows),
                "entropy": entropy.view(batch, rows), "top_tokens": top.view(batch, rows, -1),
                "top_logprobs": top_scores.view(batch, rows, -1), "logits": logits}


def main():
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--small", action="store_true", help="a toy model")
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--prompt", type=int, default=200, help="tokens that all sequences share")
    ap.add_argument("--sequences", type=int, default=4)
    ap.add_argument("--rows", type=int, default=4, help="rows of a block: a token and its drafts")
    ap.add_argument("--passes", type=int, default=4)
    ap.add_argument("--temperature", type=float, default=0.0, help="0: the likeliest tokens")
    a = ap.parse_args()
    shape = ((512, 8, 2, 64, 1024, 2000) if a.small else (5120, 40, 8, 128, 17408, 151936))
    vocab = shape[-1]
    ctx = dflash_qmm.Context(0)
    model = Decoder(ctx, a.layers, *shape, a.sequences, a.prompt, a.passes * a.rows + a.rows)
    gen = torch.Generator().manual_seed(1)
    prompt = torch.randint(0, vocab, (a.prompt,), generator=gen, dtype=torch.int32).cuda()
    first = model.ctx.token_logprobs(model.read_prompt(prompt), top_k=a.sequences)
    # the sequences start with the likeliest tokens after the prompt
    last = first[2][0].contiguous()
    starts = torch.zeros(a.sequences, dtype=torch.int32, device="cuda")
    for n in range(a.passes):
        # drafts: what the model takes after each token, the last of them replaced
        block = last[:, None]
        while block.shape[1] < a.rows:
            seen = model.verify(block, starts, top_k=1)["tokens"]
            block = torch.cat((block, seen[:, -1:]), 1)
        if a.rows > 2:
            block[:, -1] = (block[:, -1] + 1) % vocab
        if a.temperature > 0:
            u = torch.rand(block.shape, generator=gen).cuda()
            tokens, kept, chances, _ = model.sample(block, starts, u, a.temperature)
            last = tokens.gather(1, kept.long()[:, None])[:, 0]
            print(f"pass {n}: kept {kept.tolist()} of {a.rows - 1} drafts, next tokens "
                  f"{last.tolist()}, chances {[[round(v, 2) for v in c] for c in chances.tolist()]}")
            starts = starts + kept + 1
            continue
        out = model.verify(block, starts)
        at = out["accepted"].long()[:, None]
        last = out["tokens"].gather(1, at)[:, 0]
        score = out["token_logprobs"].gather(1, at)[:, 0]
        print(f"pass {n}: accepted {out['accepted'].tolist()} of {a.rows - 1} drafts, next "
              f"tokens {last.tolist()}, log probabilities "
              f"{[round(v, 2) for v in score.tolist()]}")
        starts = starts + out["accepted"] + 1
    ctx.close()


if __name__ == "__main__":
    main()
