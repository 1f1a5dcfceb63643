"""The example decoder, against a plain one that holds everything in 64 bits except what the operators' formats define: the
dequantised weights and the activations' bf16 (rounded where the example's are)."""
import os
import sys

import pytest
import torch
import torch.nn.functional as F

from if_i_could_turn_back_time_b200 import ops

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
import decode                                                     # noqa: E402

pytestmark = pytest.mark.gpu


def _plain_logits(model, tokens):
    """Logits of a whole sequence, attention over unquantised keys and values, in 64 bits."""
    w = lambda m: ops.dequantize(m.packed).double()               # noqa: E731
    x = model.embed(tokens).double()
    for layer in model.layers:
        h = F.rms_norm(x, x.shape[-1:])
        n, D, G = len(tokens), layer.dim, layer.heads // layer.kv_heads
        q = (h @ w(layer.q).T).view(n, layer.heads, D)
        k, v = ((h @ w(m).T).view(n, layer.kv_heads, D).repeat_interleave(G, 1) for m in (layer.k, layer.v))
        s = torch.einsum("qhd,khd->hqk", q, k) / D ** 0.5
        p = torch.softmax(s.masked_fill(torch.ones(n, n, device=s.device).triu(1).bool(), -torch.inf), -1)
        x = x + torch.einsum("hqk,khd->qhd", p, v).reshape(n, -1) @ w(layer.o).T
        x = x + F.silu(F.rms_norm(x, x.shape[-1:]) @ w(layer.up).T) @ w(layer.down).T
    return F.rms_norm(x, x.shape[-1:]) @ w(model.head).T


@pytest.mark.parametrize("weights,cache,kv_heads", [("gf4", "int8", 2), ("e2m1", "e4m3", 8)])
def test_prompts_and_answers(weights, cache, kv_heads):
    """Log probabilities stand within 0.1 of the plain model's: bf16 activations (2^-9 a rounding, some ten of them on the way) and
    8-bit keys and values (2^-4 and less of an element, averaged over 64) move logits of spread 0.6 by a few hundredths."""
    torch.manual_seed(0)
    model = decode.packed(decode.Decoder(2, 512, 8, kv_heads, 1024, 1000), weights)
    gen = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, 1000, (n,), generator=gen).tolist() for n in (5, 170, 1, 33)]
    answers, scored, logprobs, entropies = decode.generate(model, prompts, 4, block_size=32, cache_fmt=cache)
    assert answers.shape == (4, 4) and logprobs.shape == (4, 4, 5) and torch.isfinite(scored).all()
    at = 0
    for i, p in enumerate(prompts):
        full = torch.tensor(p + answers[i].tolist(), device="cuda")
        lp = torch.log_softmax(_plain_logits(model, full), -1)
        want = lp[:-1].gather(1, full[1:, None])[:, 0]
        assert scored[at + len(p) - 1] == 0
        assert (scored[at:at + len(p) - 1] - want[:len(p) - 1]).abs().max().item() < 0.1 if len(p) > 1 else True
        at += len(p)
        assert (logprobs[i, :, 0] - want[len(p) - 1:]).abs().max().item() < 0.1
        best = lp[len(p) - 1:-1].max(-1).values
        assert (best - want[len(p) - 1:]).max().item() < 0.2                           # the chosen one is (nearly) the strongest
        assert (entropies[i] + (lp.exp() * lp).sum(-1)[len(p) - 1:-1]).abs().max().item() < 0.1
        assert (logprobs[i].diff(dim=-1) <= 0).all()
