"""A small decoder of linear-attention and full-attention layers on the framework's operators:
W4A16 projections, RMSNorm, the gated delta rule, several-axis rotary positions with the
write into a paged cache, one-token paged attention, and the greedy lm_head.

    python examples/hybrid_decoder.py [--layers 8] [--tokens 32]

Three ragged prompts, one of them with an image's grid of tokens, are read in one packed
pass; then every sequence is continued token by token.  Random weights: what it shows is
how the calls fit together, and that both ways of reading a text agree.
"""
from __future__ import annotations

import argparse
import sys
import time
from pathlib import Path

import numpy as np
import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))
import __graft_entry__  # noqa: E402

mcv = __graft_entry__.load_package()

H, VOCAB, INNER, EPS = 1024, 4000, 3584, 1e-6
HK, HV, DL = 16, 16, 128                 # linear attention: key and value heads
HQ, HKV, DF, ROT, PAGE = 8, 2, 256, 64, 16   # full attention


def weight(rng, k, n):
    w = (rng.standard_normal((k, n)) * k ** -0.5).astype(np.float16)
    return mcv.W4A16QuantizedWeight.from_awq(*mcv.quantize_int4(w), device="cuda")


class Layer:
    def __init__(self, rng, full):
        self.full = full
        ones = torch.ones(H, dtype=torch.float16, device="cuda")
        self.norm, self.mlp_norm = ones, ones.clone()
        if full:
            self.qkv, self.o = weight(rng, H, (HQ + 2 * HKV) * DF), weight(rng, HQ * DF, H)
        else:
            self.qkv, self.o = weight(rng, H, (2 * HK + HV) * DL), weight(rng, HV * DL, H)
            self.gates = torch.from_numpy((rng.standard_normal((H, 2 * HV)) * H ** -0.5).astype(np.float16)).cuda()
            self.rate = torch.from_numpy(np.exp(rng.uniform(np.log(0.05), np.log(4), HV)).astype(np.float32)).cuda()
        self.gate, self.up, self.down = weight(rng, H, INNER), weight(rng, H, INNER), weight(rng, INNER, H)


class Decoder:
    def __init__(self, layers, sequences, max_len, seed=0):
        rng = np.random.default_rng(seed)
        self.layers = [Layer(rng, i % 4 == 3) for i in range(layers)]
        self.embedding = torch.from_numpy((rng.standard_normal((VOCAB, H)) * 0.5).astype(np.float16)).cuda()
        self.final_norm = torch.ones(H, dtype=torch.float16, device="cuda")
        self.head = weight(rng, H, -(-VOCAB // 64) * 64)
        self.freq, self.axis = mcv.rotary_axes_table(ROT, 1e7, (11, 11, 10))
        self.B, width = sequences, -(-max_len // PAGE)
        # one table for all layers, its pages dealt out in mixed order; every layer has its own caches and states
        self.table = torch.from_numpy(rng.permutation(sequences * width).astype(np.int32)).cuda().view(sequences, width)
        self.caches, self.states = {}, {}
        for i, layer in enumerate(self.layers):
            if layer.full:
                self.caches[i] = [torch.zeros(sequences * width, PAGE, HKV, DF, dtype=torch.float16, device="cuda") for _ in range(2)]
            else:
                self.states[i] = torch.zeros(sequences, HV, DL, DL, dtype=torch.float32, device="cuda")
        self.lens = torch.zeros(sequences, dtype=torch.int32, device="cuda")         # tokens each sequence holds

    def run(self, tokens, positions, seq, at, cu):
        """Hidden rows [T, H] of packed tokens: their sequence, place in it and positions [3, T].
        cu: where the sequences' tokens begin; None: one token for each sequence in order."""
        T = len(tokens)
        x = self.embedding[tokens]
        slots = self.table[seq, at // PAGE].long() * PAGE + at % PAGE
        rows_table, rows_len = (self.table, (at + 1).int()) if cu is None else (self.table[seq], (at + 1).int())
        for i, layer in enumerate(self.layers):
            qkv = mcv.matmul_w4a16(mcv.rms_norm(x, layer.norm, EPS), layer.qkv)
            if layer.full:
                q, k, v = (t.view(T, -1, DF) for t in qkv.split((HQ * DF, HKV * DF, HKV * DF), 1))
                kc, vc = self.caches[i]
                q = mcv.rotary_axes_cached(q, k, v, positions, self.freq, self.axis, kc, vc, slots)
                y = mcv.paged_attention_decode(q, kc, vc, rows_table, rows_len)      # a prompt: each token a row of its own
            else:
                qkv = torch.nn.functional.silu(qkv)
                q, k, v = (t.view(T, -1, DL) for t in qkv.split((HK * DL, HK * DL, HV * DL), 1))
                a, b = (x @ layer.gates).float().chunk(2, 1)
                g, beta = (-layer.rate * torch.nn.functional.softplus(a - 2)), torch.sigmoid(b).contiguous()
                state = self.states[i]
                if cu is None:
                    y, _ = mcv.gated_delta_rule_step(q, k, v, g, beta, state, normalize=True)
                else:
                    y, _ = mcv.gated_delta_rule(q, k, v, g, beta, state, cu_seqlens=cu, normalize=True, state_out=state)
            x = x + mcv.matmul_w4a16(y.reshape(T, -1), layer.o)
            h = mcv.rms_norm(x, layer.mlp_norm, EPS)
            x = x + mcv.matmul_w4a16(mcv.mlp_gate_up_silu_w4a16(h, layer.gate, layer.up), layer.down)
        return x

    def logits(self, x):
        return mcv.matmul_w4a16(mcv.rms_norm(x, self.final_norm, EPS), self.head)[:, :VOCAB].contiguous()

    def read(self, prompts, positions):
        """Whole prompts at once, from empty states and caches; the last rows' logits."""
        n = torch.tensor([len(p) for p in prompts])
        cu = torch.cat((torch.zeros(1, dtype=torch.int64), n.cumsum(0))).int().cuda()
        seq = torch.repeat_interleave(torch.arange(self.B), n).cuda()
        at = torch.cat([torch.arange(int(m)) for m in n]).cuda()
        for s in self.states.values():
            s.zero_()
        self.lens.copy_(n)
        x = self.run(torch.cat(prompts).cuda(), torch.cat(positions, 1).contiguous().cuda(), seq, at, cu)
        return self.logits(x[cu[1:].long() - 1].contiguous())

    def step(self, tokens, positions):
        """One more token for every sequence."""
        at = self.lens.long()
        x = self.run(tokens, positions, torch.arange(self.B, device="cuda"), at, None)
        self.lens += 1
        return self.logits(x)


def text(n, start=0):
    return (start + torch.arange(n)).expand(3, n)


def prompts(gen):
    """Texts of 37 and 5 tokens, and one of 20 with an image of 8 x 6 behind it; the position each goes on with."""
    tokens = [torch.randint(0, VOCAB, (n,), generator=gen) for n in (37, 5, 20 + 48)]
    h, w = torch.arange(48) // 6, torch.arange(48) % 6
    image = torch.stack((torch.zeros(48, dtype=torch.int64), h, w)) + 20
    return tokens, [text(37), text(5), torch.cat((text(20), image), 1)], torch.tensor([37, 5, 28])


def main(layers=8, steps=32, seed=0):
    gen = torch.Generator().manual_seed(seed)
    tokens, positions, after = prompts(gen)
    model = Decoder(layers, len(tokens), max(map(len, tokens)) + steps + 1, seed)
    logits = model.read(tokens, positions)
    after = after.cuda()
    said = []
    torch.cuda.synchronize()
    start = time.perf_counter()
    for i in range(steps):
        token = mcv.argmax_last_dim(logits)
        said.append(token)
        logits = model.step(token, (after + i).expand(3, -1).contiguous())
    torch.cuda.synchronize()
    took = (time.perf_counter() - start) / steps
    # the same tokens read at once end where the steps ended
    more = torch.stack(said, 1).cpu()
    whole = model.read([torch.cat((t, m)) for t, m in zip(tokens, more)],
                       [torch.cat((p, text(steps, int(n))), 1) for p, n in zip(positions, after.tolist())])
    apart = float((whole.double() - logits.double()).norm() / logits.double().norm())
    return more, took, apart


if __name__ == "__main__":
    args = argparse.ArgumentParser()
    args.add_argument("--layers", type=int, default=8)
    args.add_argument("--tokens", type=int, default=32)
    a = args.parse_args()
    more, took, apart = main(a.layers, a.tokens)
    for row in more.tolist():
        print(" ".join(map(str, row[:16])), "...")
    print(f"{took * 1e3:.2f} ms a step of {len(more)} sequences and {a.layers} layers; read at once, the logits are {apart:.1e} apart")
