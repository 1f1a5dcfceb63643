"""A small decoder of packed 4-bit layers that answers with alternatives: the prompt goes through in one pass, then token by token.

Its matrices are ``JenksQuantLinear`` layers, what its attention reads lies in a ``KVCache`` of 8 bits per layer, and every
position's log probability, entropy and strongest alternatives come from ``ops.token_logprobs``.  Weights are random: what
it shows is how the calls fit together, with sequences of different lengths in one batch.

    python examples/decode.py --layers 2 --hidden 512 --heads 8 --kv-heads 2 --new 8
"""
import argparse
import os
import sys

import torch
import torch.nn as nn
import torch.nn.functional as F

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import if_i_could_turn_back_time_b200 as jq                   # noqa: E402
from if_i_could_turn_back_time_b200 import ops                # noqa: E402


class Layer(nn.Module):
    def __init__(self, hidden, heads, kv_heads, ffn):
        super().__init__()
        self.heads, self.kv_heads, self.dim = heads, kv_heads, hidden // heads
        self.q, self.o = nn.Linear(hidden, hidden, bias=False), nn.Linear(hidden, hidden, bias=False)
        self.k, self.v = (nn.Linear(hidden, kv_heads * self.dim, bias=False) for _ in range(2))
        self.up, self.down = nn.Linear(hidden, ffn, bias=False), nn.Linear(ffn, hidden, bias=False)

    def forward(self, x, cache, table, lengths, starts, max_new):
        h = F.rms_norm(x, x.shape[-1:])
        q = self.q(h).view(-1, self.heads, self.dim)
        k, v = self.k(h).view(-1, self.kv_heads, self.dim), self.v(h).view(-1, self.kv_heads, self.dim)
        cache.append(k, v, table, lengths, starts, max_new)
        x = x + self.o(cache.attend(q, table, lengths, starts, max_new).view(x.shape))
        return x + self.down(F.silu(self.up(F.rms_norm(x, x.shape[-1:]))))


class Decoder(nn.Module):
    def __init__(self, layers, hidden, heads, kv_heads, ffn, vocab):
        super().__init__()
        self.embed = nn.Embedding(vocab, hidden)
        self.layers = nn.ModuleList(Layer(hidden, heads, kv_heads, ffn) for _ in range(layers))
        self.head = nn.Linear(hidden, vocab, bias=False)

    def forward(self, tokens, caches, table, lengths, starts, max_new):
        """Logits of the new tokens [tokens], which the sequences' lengths count already."""
        x = self.embed(tokens)
        for layer, cache in zip(self.layers, caches):
            x = layer(x, cache, table, lengths, starts, max_new)
        return self.head(F.rms_norm(x, x.shape[-1:]))


def packed(model, fmt="gf4"):
    """The model with every Linear as packed 4-bit weights, on the GPU in bf16."""
    model = jq.quantize_module(model, 4, fmt=fmt, group_size=128 if fmt == "gf4" else 32).to("cuda")
    for m in model.modules():
        if isinstance(m, jq.JenksQuantLinear):
            m.commit()
    model.embed.to(torch.bfloat16)
    return model


@torch.no_grad()
def generate(model, prompts, new, *, block_size=64, cache_fmt="int8", top=5):
    """Answers `new` tokens to each prompt (lists of token numbers), always the strongest.  Returns (answers [sequences, new], the
    log probability of every prompt token given those before it, log probabilities and entropies of the answers)."""
    layer = model.layers[0]
    S, longest = len(prompts), max(map(len, prompts)) + new
    width = -(-longest // block_size)
    caches = [jq.KVCache.empty(S * width, layer.kv_heads, layer.dim, block_size=block_size, fmt=cache_fmt) for _ in model.layers]
    table = torch.arange(S * width, dtype=torch.int32, device="cuda").view(S, width)
    counts = [len(p) for p in prompts]
    lengths = torch.tensor(counts, dtype=torch.int32, device="cuda")
    starts = torch.tensor([0] + counts, device="cuda").cumsum(0).int()
    tokens = torch.tensor(sum(prompts, []), device="cuda")

    logits = model(tokens, caches, table, lengths, starts, max(counts))
    following = torch.cat([tokens[1:], tokens[:1]])
    following[starts[1:].long() - 1] = -1                       # (behind a prompt's last token there is none: 0)
    scored = ops.token_logprobs(logits, following, top=0).logprob
    logits = logits[starts[1:].long() - 1]
    answers, logprobs, entropies = [], [], []
    for _ in range(new):
        found = ops.token_logprobs(logits, torch.full((S,), -1, device="cuda"), top=top)
        answers.append(found.top_tokens[:, 0])
        logprobs.append(found.top_logprobs)
        entropies.append(found.entropy)
        lengths += 1
        logits = model(answers[-1], caches, table, lengths, None, 1)
    if ops.check_status(raise_on_error=False):
        raise RuntimeError("a device-side wait gave up")
    return torch.stack(answers, 1), scored, torch.stack(logprobs, 1), torch.stack(entropies, 1)


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, default in (("layers", 2), ("hidden", 512), ("heads", 8), ("kv-heads", 2), ("ffn", 1024), ("vocab", 4000), ("new", 8)):
        ap.add_argument("--" + name, type=int, default=default)
    ap.add_argument("--weights", choices=("gf4", "e2m1"), default="gf4")
    ap.add_argument("--cache", choices=("int8", "e4m3"), default="int8")
    a = ap.parse_args(argv)
    torch.manual_seed(0)
    model = packed(Decoder(a.layers, a.hidden, a.heads, a.kv_heads, a.ffn, a.vocab), a.weights)
    gen = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, a.vocab, (n,), generator=gen).tolist() for n in (5, 70, 1, 33)]
    answers, scored, logprobs, entropies = generate(model, prompts, a.new, cache_fmt=a.cache)
    at = 0
    for i, p in enumerate(prompts):
        print(f"prompt of {len(p)} tokens, sum of log probabilities {scored[at:at + len(p)].sum().item():.2f}; answer "
              f"{answers[i].tolist()}, log probabilities {[round(v, 3) for v in logprobs[i, :, 0].tolist()]}, "
              f"entropies {[round(v, 3) for v in entropies[i].tolist()]}")
        at += len(p)
    return answers, scored, logprobs, entropies


if __name__ == "__main__":
    main()
