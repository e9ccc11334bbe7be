"""Decoding that verifies trees of drafted tokens, on int8 weights and an int8 key/value cache.

A step drafts continuations of the text (here: what followed the same words before, a tree where they differ), runs all of them
through the decoder in one pass and keeps the longest path that the decoder itself would have chosen:

    rows      the newest token and its drafted descendants, each at the position of its depth
    linears   symmetric_quant_matmul on int8 weights, SwiGLU and residuals in its epilogue
    cache     quantized_cache_append rotates the rows' queries and keys and writes keys and values behind the text
    attention quantized_cache_attention: a row sees the text and, by the mask, its ancestors
    choice    token_log_probs: the log probabilities of every row's drafted children and of its best token
    keeping   the accepted path's rows move to the front (quantized_cache_read, quantized_cache_append)

The pass has a fixed number of rows and everything that changes is on the device, so it is captured once and replayed
(CudaGraph).  The decoder is bench_decoder.py's, with random weights.

    python examples/tree_decoding.py [--full] [--tokens N] [--rows W]
"""
from __future__ import annotations

import argparse
import json
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import bench_decoder  # noqa: E402
import hidet_b200  # noqa: E402
from hidet_b200.quant import interleave_gate_up, symmetric_quant_matmul as linear  # noqa: E402

PAGE = 64


def quantized(*weights):
    """Weights of linears [out, in], side by side: int8 [in, out] and its scales."""
    return hidet_b200.symmetric_quantize(torch.cat([w.detach() for w in weights]).t().contiguous(), 'int8', dims=0)


class QuantizedDecoder:
    """bench_decoder.Decoder with int8 linears, an int8 embedding table and a quantized, paged cache for one sequence."""

    def __init__(self, model: bench_decoder.Decoder, positions: int):
        cfg, device = model.cfg, model.norm.device
        self.heads, self.dim, self.norm = cfg.heads, cfg.hidden // cfg.heads, model.norm
        self.embedding = hidet_b200.symmetric_quantize(model.embed.weight.detach(), 'int8', dims=-1)
        self.layers = []
        for layer in model.layers:
            gate, up = quantized(layer.gate.weight), quantized(layer.up.weight)
            self.layers.append((layer.n1, quantized(layer.q.weight, layer.k.weight, layer.v.weight), quantized(layer.o.weight), layer.n2,
                                (interleave_gate_up(gate[0], up[0]), interleave_gate_up(gate[1], up[1])), quantized(layer.down.weight)))
        self.head = quantized(model.head.weight)
        self.table = hidet_b200.rotary_table(positions, self.dim, device=device)
        pages = -(-positions // PAGE)
        self.caches = [hidet_b200.quantized_cache(pages, cfg.heads, self.dim, PAGE, device=device) for _ in self.layers]
        self.pages = torch.arange(pages, dtype=torch.int32, device=device)[None]  # of the one sequence, in order: its slots are its positions

    def __call__(self, ids, positions, slots, length, mask=None):
        """Logits of the rows ids [t].  length [1]: what is in the cache, these rows included."""
        rms = bench_decoder.rms
        x = hidet_b200.symmetric_dequantize_take(*self.embedding, ids)
        for (n1, qkv, o, n2, gate_up, down), cache in zip(self.layers, self.caches):
            q, k, v = linear(rms(x, n1), *qkv).view(len(ids), 3, self.heads, self.dim).unbind(1)
            q = hidet_b200.quantized_cache_append(cache, k, v, slots, q=q, positions=positions, table=self.table, layout='interleaved')
            a = hidet_b200.quantized_cache_attention(q[None], cache, self.pages, length, mask=mask)
            x = linear(a.flatten(2)[0], *o, residual=x)
            x = linear(linear(rms(x, n2), *gate_up, activation='silu_mul'), *down, residual=x)
        return linear(rms(x, self.norm), *self.head)

    def move(self, source, target):
        """Rows of the cache to other slots.  Codes stay as they are: a row's largest is 127, whatever its scale."""
        for cache in self.caches:
            hidet_b200.quantized_cache_append(cache, *hidet_b200.quantized_cache_read(cache, source, torch.float32), target)


def followers(text, rows, depth=6, branches=4):
    """Continuations of the text that were seen in it: after its last two tokens, and then after its last."""
    found = []
    for n in (2, 1):
        for at in range(len(text) - n, n - 1, -1):
            if text[at - n:at] == text[-n:] and text[at:at + depth] not in found:
                found.append(text[at:at + depth])
            if len(found) == branches:
                return found
    return found


def tree_of(newest, continuations, rows):
    """(tokens, parents) of a tree of at most `rows` nodes with the newest token at its root."""
    tokens, parents, children = [newest], [-1], [{}]
    for path in continuations:
        at = 0
        for token in path:
            if token not in children[at]:
                if len(tokens) == rows:
                    break
                children[at][token] = len(tokens)
                tokens.append(token)
                parents.append(at)
                children.append({})
            at = children[at][token]
    return tokens, parents


class TreeDecoding:
    """Greedy decoding of one sequence by passes over `rows` rows."""

    def __init__(self, model: bench_decoder.Decoder, positions: int, rows: int = 16, draft=followers):
        self.decoder, self.rows, self.draft = QuantizedDecoder(model, positions + rows), rows, draft
        self.device = model.norm.device
        inputs = [torch.zeros(rows, dtype=torch.int64, device=self.device), torch.zeros(rows, dtype=torch.int64, device=self.device),
                  torch.full((rows,), -1, dtype=torch.int64, device=self.device), torch.full((1,), rows, dtype=torch.int32, device=self.device),
                  torch.zeros((rows, rows), dtype=torch.bool, device=self.device), torch.zeros((rows, rows), dtype=torch.int64, device=self.device)]
        self.graph = hidet_b200.CudaGraph(lambda: inputs, lambda x: self.verify(*x), ref_objs=[self.decoder])

    def verify(self, ids, positions, slots, length, mask, candidates):
        """Of every row: the log probabilities of the candidates, and its best token's with the token."""
        log_probs, _, best, token = hidet_b200.token_log_probs(self.decoder(ids, positions, slots, length, mask), candidates, top=1)
        return [log_probs, best, token]

    def prompt(self, ids):
        """The prompt's pass; the first token and its log probability."""
        at = torch.arange(len(ids), device=self.device)
        logits = self.decoder(ids, at, at, torch.tensor([len(ids)], dtype=torch.int32, device=self.device))
        _, _, best, token = hidet_b200.token_log_probs(logits[-1:], ids[-1:], top=1)
        return token.item(), best.item()

    def generate(self, prompt, count: int, slack: float = 0.0):
        """(tokens, their log probabilities, passes).  A drafted token is taken where its log probability is the best one's, or less by at most `slack`."""
        text = prompt.tolist()
        token, log_prob = self.prompt(prompt)
        text.append(token)
        tokens, log_probs, passes = [token], [log_prob], 0
        while len(tokens) < count:
            base = len(text) - 1  # what the cache holds; the newest token is not in it yet
            ids, parents = tree_of(text[-1], self.draft(text, self.rows), self.rows)
            n = len(ids)
            depth, sees, children = [0] * n, [[False] * self.rows for _ in range(self.rows)], [[] for _ in range(n)]
            for i in range(n):
                if i:
                    depth[i] = depth[parents[i]] + 1
                    sees[i] = list(sees[parents[i]])
                    children[parents[i]].append(i)
                sees[i][i] = True
            candidates = torch.zeros((self.rows, self.rows), dtype=torch.int64)
            for i, c in enumerate(children):
                candidates[i, :len(c)] = torch.tensor([ids[j] for j in c], dtype=torch.int64)
            pad = self.rows - n  # rows without a token: no slot, nothing seen of them
            step = [torch.tensor(ids + [0] * pad), torch.tensor([base + d for d in depth] + [0] * pad), torch.tensor([base + i for i in range(n)] + [-1] * pad),
                    torch.tensor([base + self.rows], dtype=torch.int32), torch.tensor(sees), candidates]
            of_children, best, choice = (x.tolist() for x in self.graph.run_async([x.to(self.device) for x in step]))
            passes += 1
            path = [0]
            while True:
                at = path[-1]
                taken = max(range(len(children[at])), key=lambda j: of_children[at][j], default=None)
                if taken is None or not of_children[at][taken] >= best[at][0] - slack:
                    break
                path.append(children[at][taken])
                tokens.append(ids[path[-1]])
                log_probs.append(of_children[at][taken])
            tokens.append(choice[path[-1]][0])
            log_probs.append(best[path[-1]][0])
            text += tokens[len(text) - len(prompt):]
            moved = [(base + i, base + to) for to, i in enumerate(path) if i != to]
            if moved:
                source, target = torch.tensor(moved, device=self.device).unbind(1)
                self.decoder.move(source, target)
        return tokens[:count], log_probs[:count], passes


def main(argv=None):
    parser = argparse.ArgumentParser()
    parser.add_argument('--full', action='store_true', help='the 7B-shaped decoder (a small one otherwise)')
    parser.add_argument('--tokens', type=int, default=96)
    parser.add_argument('--rows', type=int, default=16)
    args = parser.parse_args(argv)
    cfg = bench_decoder.LLAMA_7B if args.full else bench_decoder.SMALL
    torch.manual_seed(7)
    with torch.device('cuda'):
        model = bench_decoder.Decoder(cfg).half().eval()
    prompt = torch.randint(0, cfg.vocab, (cfg.prompt,), device='cuda', generator=torch.Generator('cuda').manual_seed(7))
    result = {}
    with torch.no_grad():
        for rows in (1, args.rows):
            decoding = TreeDecoding(model, cfg.prompt + args.tokens, rows)
            decoding.generate(prompt, 4)
            start = time.perf_counter()
            tokens, log_probs, passes = decoding.generate(prompt, args.tokens)
            result['rows_{}'.format(rows)] = {'tokens': len(tokens), 'passes': passes, 'ms_per_token': round((time.perf_counter() - start) * 1e3 / len(tokens), 3),
                                              'mean_log_prob': round(sum(log_probs) / len(log_probs), 4)}
            del decoding
    print(json.dumps(result))
    return result


if __name__ == '__main__':
    main()
