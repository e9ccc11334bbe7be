"""Decoding with a layer of experts in every block, on int8 weights: a prompt on int8 tokens, then a token at a time.

    prompt    quantize_tokens behind the norm, symmetric_quant_matmul_i8 (int8 products) with the residual in its epilogue
    a token   symmetric_quant_matmul (weight-only: reading the weight is all the time)
    experts   route_tokens and mixture_of_experts, the layer's input its residual, in the input's place
    cache     quantized_cache_append and quantized_cache_attention
    choice    token_log_probs

The same int8 weights and scales serve both kinds of linears.  The pass of a token is captured once and replayed (CudaGraph).  Weights are random.

    python examples/expert_decoding.py [--prompt N] [--tokens N] [--large]
"""
from __future__ import annotations

import argparse
import json
import os
import sys
import time
from dataclasses import dataclass

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import hidet_b200  # noqa: E402

PAGE = 64
EPS = 1e-5


@dataclass
class Config:
    hidden: int = 256
    heads: int = 4
    layers: int = 2
    experts: int = 8
    top: int = 2
    inner: int = 384
    vocab: int = 512


LARGE = Config(hidden=2048, heads=16, layers=8, experts=64, top=6, inner=1408, vocab=32000)


def random_weights(cfg: Config, device='cuda', dtype=torch.float16, seed=11):
    """Float weights: embedding, head, and for every layer its two norms, qkv and o [in, out], router [experts, hidden], gate_up [experts, 2 inner, hidden] and down [experts, hidden, inner]."""
    gen = torch.Generator(device=device).manual_seed(seed)

    def normal(*shape, std):
        return (torch.randn(shape, generator=gen, device=device) * std).to(dtype)

    h, i = cfg.hidden, cfg.inner
    layers = [dict(n1=1 + normal(h, std=0.1), qkv=normal(h, 3 * h, std=h ** -0.5), o=normal(h, h, std=h ** -0.5), n2=1 + normal(h, std=0.1), router=normal(cfg.experts, h, std=2 * h ** -0.5),
                   gate_up=normal(cfg.experts, 2 * i, h, std=h ** -0.5), down=normal(cfg.experts, h, i, std=i ** -0.5)) for _ in range(cfg.layers)]
    return dict(embedding=normal(cfg.vocab, h, std=1.0), norm=1 + normal(h, std=0.1), head=normal(h, cfg.vocab, std=h ** -0.5), layers=layers)


def rms(x, weight):
    y = x.float()
    return (y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * weight.float()).to(x.dtype)


class ExpertDecoder:
    """int8 linears and experts, and a quantized cache for one sequence of up to `positions`."""

    def __init__(self, cfg: Config, weights, positions: int):
        self.cfg, self.dim = cfg, cfg.hidden // cfg.heads
        device = weights['head'].device
        self.embedding, self.norm, self.head = weights['embedding'], weights['norm'], hidet_b200.symmetric_quantize(weights['head'], 'int8', dims=0)
        self.layers = []
        for w in weights['layers']:
            self.layers.append(dict(w, qkv=hidet_b200.symmetric_quantize(w['qkv'], 'int8', dims=0), o=hidet_b200.symmetric_quantize(w['o'], 'int8', dims=0),
                                    gate_up=hidet_b200.symmetric_quantize(w['gate_up'], 'int8', dims=-1), down=hidet_b200.symmetric_quantize(w['down'], 'int8', dims=-1)))
        pages = -(-positions // PAGE)
        self.table = hidet_b200.rotary_table(pages * PAGE, self.dim, device=device)
        self.caches = [hidet_b200.quantized_cache(pages, cfg.heads, self.dim, PAGE, device=device) for _ in self.layers]
        self.pages = torch.arange(pages, dtype=torch.int32, device=device)[None]  # of the one sequence, in order: its slots are its positions

    def linear(self, x, weight, norm=None, residual=None):
        """x (behind an RMS norm) times an int8 weight: on int8 tokens where there are many, on float16 ones where the weight's bytes are the time."""
        if x.shape[0] > 64:
            return hidet_b200.symmetric_quant_matmul_i8(*hidet_b200.quantize_tokens(x, norm, EPS), *weight, residual=residual)
        return hidet_b200.symmetric_quant_matmul(x if norm is None else rms(x, norm), *weight, residual=residual)

    def __call__(self, ids, positions, length):
        """Logits of the rows ids [t] at positions [t]; length [1]: what is in the cache, these rows included."""
        cfg = self.cfg
        x = self.embedding[ids]
        for w, cache in zip(self.layers, self.caches):
            q, k, v = self.linear(x, w['qkv'], w['n1']).view(len(ids), 3, cfg.heads, self.dim).unbind(1)
            q = hidet_b200.quantized_cache_append(cache, k, v, positions, q=q, positions=positions, table=self.table)
            a = hidet_b200.quantized_cache_attention(q[None], cache, self.pages, length)
            x = self.linear(a.flatten(2)[0], w['o'], residual=x)
            y = rms(x, w['n2'])
            experts, weights = hidet_b200.route_tokens(y, w['router'], cfg.top)
            x = hidet_b200.mixture_of_experts(y, experts, weights, *w['gate_up'], *w['down'], residual=x, out=x)
        return self.linear(x, self.head, self.norm)


class Decoding:
    """Greedy decoding of one sequence: the prompt in one pass, then replays of a token's."""

    def __init__(self, cfg: Config, weights, positions: int):
        self.decoder = ExpertDecoder(cfg, weights, positions)
        device = weights['head'].device
        inputs = [torch.zeros(1, dtype=torch.int64, device=device), torch.zeros(1, dtype=torch.int64, device=device), torch.ones(1, dtype=torch.int32, device=device)]
        self.graph = hidet_b200.CudaGraph(lambda: inputs, lambda x: self.step(*x), ref_objs=[self.decoder])

    def step(self, ids, positions, length):
        _, entropy, best, token = hidet_b200.token_log_probs(self.decoder(ids, positions, length), ids, top=1)
        return [token[:, 0], best, entropy]

    def generate(self, prompt, count: int):
        """(tokens, their log probabilities)"""
        at = torch.arange(len(prompt), device=prompt.device)
        logits = self.decoder(prompt, at, torch.tensor([len(prompt)], dtype=torch.int32, device=prompt.device))
        _, _, best, token = hidet_b200.token_log_probs(logits[-1:], prompt[-1:], top=1)
        tokens, log_probs = [token[0, 0].clone()], [best[0, 0].clone()]
        for n in range(len(prompt), len(prompt) + count - 1):
            position = torch.tensor([n], device=prompt.device)
            token, best, _ = self.graph.run_async([tokens[-1][None], position, (position + 1).int()])
            tokens.append(token[0].clone())
            log_probs.append(best[0, 0].clone())
        return torch.stack(tokens).tolist(), torch.stack(log_probs).tolist()


def main(argv=None):
    parser = argparse.ArgumentParser()
    parser.add_argument('--prompt', type=int, default=200)
    parser.add_argument('--tokens', type=int, default=64)
    parser.add_argument('--large', action='store_true', help='64 experts of 2048 x 1408 in 8 layers (8 small ones in 2 otherwise)')
    args = parser.parse_args(argv)
    cfg = LARGE if args.large else Config()
    weights = random_weights(cfg)
    prompt = torch.randint(0, cfg.vocab, (args.prompt,), device='cuda', generator=torch.Generator('cuda').manual_seed(5))
    with torch.no_grad():
        decoding = Decoding(cfg, weights, args.prompt + args.tokens)
        decoding.generate(prompt, 4)
        start = time.perf_counter()
        tokens, log_probs = decoding.generate(prompt, args.tokens)
        ms = (time.perf_counter() - start) * 1e3
    result = {'prompt': args.prompt, 'tokens': len(tokens), 'ms_per_token': round(ms / len(tokens), 3), 'mean_log_prob': round(sum(log_probs) / len(log_probs), 4)}
    print(json.dumps(result))
    return result


if __name__ == '__main__':
    main()
