"""examples/expert_decoding.py: the linears on int8 tokens and the layers of experts as a decoder uses them, against the same decoder in float32."""
import os
import sys

import pytest
import torch

from conftest import ROOT

sys.path.insert(0, os.path.join(ROOT, 'examples'))
import expert_decoding as example  # noqa: E402

import hidet_b200
from hidet_b200 import ffi

pytestmark = pytest.mark.gpu


def plain_logits(cfg, weights, ids):
    """The whole text at once, in float32 and with float weights."""
    dim, n = cfg.hidden // cfg.heads, len(ids)
    x = weights['embedding'][ids].float()
    table = hidet_b200.rotary_table(n, dim, device=ids.device)
    cos, sin = table[:, None, :dim // 2], table[:, None, dim // 2:]

    def rotated(v):
        a, b = v[..., :dim // 2], v[..., dim // 2:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

    def rms(v, w):
        return v * torch.rsqrt(v.square().mean(-1, keepdim=True) + example.EPS) * w.float()

    for w in weights['layers']:
        q, k, v = (rms(x, w['n1']) @ w['qkv'].float()).view(n, 3, cfg.heads, dim).unbind(1)
        s = torch.einsum('qhd,khd->hqk', rotated(q), rotated(k)) * dim ** -0.5
        s = s.masked_fill(torch.ones(n, n, dtype=torch.bool, device=ids.device).triu(1), -float('inf'))
        x = x + torch.einsum('hqk,khd->qhd', s.softmax(-1), v).flatten(1) @ w['o'].float()
        y = rms(x, w['n2'])
        p, chosen = (y @ w['router'].float().t()).softmax(-1).topk(cfg.top, -1)
        p = p / p.sum(-1, keepdim=True)
        for e in range(cfg.experts):
            g = y @ w['gate_up'][e].float().t()
            h = torch.nn.functional.silu(g[:, 0::2]) * g[:, 1::2]
            x = x + torch.where(chosen == e, p, 0.0).sum(-1, keepdim=True) * (h @ w['down'][e].float().t())
    return rms(x, weights['norm']) @ weights['head'].float()


@pytest.mark.parametrize('tokens', [150, 40])
def test_prompt_and_steps_against_float(tokens):
    """150 tokens go through the int8 products, 40 through the weight-only ones.  A code is off by up to half a step of 1/127 of its row's largest, about 1 % of its typical element, in
    weights and tokens; four products a layer and two layers make some 5 % of the logits' size, and a token near a border between experts, which goes elsewhere, more: half of the tokens
    stay below 10 % and all together below 30 %."""
    cfg = example.Config()
    weights = example.random_weights(cfg)
    ids = torch.randint(0, cfg.vocab, (tokens + 5,), device='cuda', generator=torch.Generator('cuda').manual_seed(3))
    decoder = example.ExpertDecoder(cfg, weights, tokens + 5)
    at = torch.arange(tokens + 5, device='cuda')
    with torch.no_grad():
        got = [decoder(ids[:tokens], at[:tokens], torch.tensor([tokens], dtype=torch.int32, device='cuda'))]
        for n in range(tokens, tokens + 5):
            got.append(decoder(ids[n:n + 1], at[n:n + 1], torch.tensor([n + 1], dtype=torch.int32, device='cuda')))
        want = plain_logits(cfg, weights, ids)
    error = (torch.cat(got).float() - want).square().mean(-1).sqrt() / want.square().mean(-1).sqrt()
    assert error.median() < 0.10 and error.square().mean().sqrt() < 0.30
    assert ffi.func('b200q_check_status')() == ffi.OK


def test_replayed_steps_are_the_steps():
    """The captured pass gives what the eager one gives, token for token."""
    cfg = example.Config()
    weights = example.random_weights(cfg)
    prompt = torch.randint(0, cfg.vocab, (100,), device='cuda', generator=torch.Generator('cuda').manual_seed(4))
    with torch.no_grad():
        tokens, log_probs = example.Decoding(cfg, weights, 130).generate(prompt, 20)
        decoder = example.ExpertDecoder(cfg, weights, 130)
        at = torch.arange(130, device='cuda')
        logits = decoder(prompt, at[:100], torch.tensor([100], dtype=torch.int32, device='cuda'))[-1]
        for n, (token, log_prob) in enumerate(zip(tokens, log_probs)):
            assert int(logits.argmax()) == token and abs(torch.log_softmax(logits.float(), -1)[token].item() - log_prob) < 1e-4
            logits = decoder(torch.tensor([token], device='cuda'), at[100 + n:101 + n], torch.tensor([101 + n], dtype=torch.int32, device='cuda'))[0]


def test_the_example_runs(capsys):
    result = example.main(['--prompt', '70', '--tokens', '8'])
    assert result['tokens'] == 8 and result['mean_log_prob'] < 0
