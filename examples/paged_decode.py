"""Serving steps of one attention layer on a paged MXFP4 cache.

A layer of SmolVLA's decoder size (hidden 960, 15 query heads on 5 K/V heads
of 64) with MXFP4 projections serves ragged requests: a step takes new tokens
of every request, a prompt's or one each, in

    hb_kv_plan -> hb_encode_mxint8 -> hb_linear (QKV) -> hb_norm_rope
    -> hb_kv_append -> hb_kv_attention -> hb_encode_mxint8 -> hb_linear (O)

on one stream: lengths, free pages and block tables stay on the device between
steps (only hb_encode_mxint8 waits, for its flag of bad input).

    python examples/paged_decode.py [--requests 8] [--steps 32]
"""
from __future__ import annotations

import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import hotarubi_amd as hb  # noqa: E402

HIDDEN, Q_HEADS, KV_HEADS, DIM, PAGE = 960, 15, 5, 64, 32
DEV = "cuda"


def _ints(*shape, fill=0):
    return torch.full(shape, fill, dtype=torch.int32, device=DEV)


class Linear:
    """An MXFP4 layer [n][k] of random weights, in the words hb_linear takes."""

    def __init__(self, n: int, k: int, gen, ctx):
        self.n, self.kb = n, k // 32
        codes = torch.randint(0, 16, (n, k), generator=gen, device=DEV, dtype=torch.int32)
        scales = torch.full((n, self.kb), 119, dtype=torch.uint8, device=DEV)
        self.words = torch.empty((n // 8 * self.kb, 144), dtype=torch.uint8, device=DEV)
        hb.mxfp4_canonical(codes.to(torch.uint8), scales, n, k, n, self.words, ctx=ctx)

    def __call__(self, x, ctx):
        rows, k = x.shape
        a = torch.empty((-(-rows // 4) * self.kb, 144), dtype=torch.uint8, device=DEV)
        out = torch.empty((rows, self.n), device=DEV)
        hb.encode_mxint8(x, rows, k, a, ctx=ctx)
        hb.linear(ctx, sync=False, a=a, planes=[self.words], modes=[0], c=out, m=rows, n=self.n,
                  kb_total=self.kb, mode=hb.FAST)
        return out


class Layer:
    """The attention layer and its cache for up to `requests` requests."""

    def __init__(self, requests: int, pages: int, most: int, ctx, seed: int = 0):
        gen = torch.Generator(device=DEV).manual_seed(seed)
        self.ctx, self.most = ctx, most
        self.qkv = Linear((Q_HEADS + 2 * KV_HEADS) * DIM, HIDDEN, gen, ctx)
        self.o = Linear(HIDDEN, Q_HEADS * DIM, gen, ctx)
        self.gamma = 1 + 0.1 * torch.randn((2, DIM), generator=gen, device=DEV)
        self.inv_freq = 10000.0 ** -(torch.arange(DIM // 2, device=DEV, dtype=torch.float64)
                                     / (DIM // 2))
        self.cache = torch.zeros(hb.kv_cache_shape(pages, KV_HEADS, PAGE, DIM), dtype=torch.uint8,
                                 device=DEV)
        self.free = torch.arange(pages, dtype=torch.int32, device=DEV)
        self.free_count = _ints(1, fill=pages)
        self.table = _ints(requests, -(-most // PAGE), fill=-1)
        self.lens = _ints(requests)
        self.cu, self.kv_lens, self.status = _ints(requests + 1), _ints(requests), _ints(2)

    def step(self, x, new, max_new: int):
        """x [tokens][HIDDEN]: new[b] (int32, on the device, at most max_new)
        tokens of each request, one request after another."""
        tokens, ctx = x.shape[0], self.ctx
        slots, positions = _ints(tokens), _ints(tokens)
        hb.kv_plan(lens=self.lens, new_tokens=new, free_pages=self.free,
                   free_count=self.free_count, table=self.table, page_size=PAGE, cu=self.cu,
                   kv_lens=self.kv_lens, slots=slots, positions=positions, status=self.status,
                   ctx=ctx, sync=False)
        rows = self.qkv(x, ctx).view(tokens, Q_HEADS + 2 * KV_HEADS, DIM)
        q, k, v = rows.split([Q_HEADS, KV_HEADS, KV_HEADS], 1)
        hb.norm_rope(q=q, k=k, q_out=q, k_out=k, positions=positions, inv_freq=self.inv_freq,
                     gamma_q=self.gamma[0], gamma_k=self.gamma[1], ctx=ctx, sync=False)
        hb.kv_append(k=k, v=v, slots=slots, cache=self.cache, ctx=ctx, sync=False)
        out = torch.empty((tokens, Q_HEADS, DIM), device=DEV)
        hb.kv_attention(q=q, out=out, cache=self.cache, table=self.table, cu=self.cu,
                        kv_lens=self.kv_lens, max_new=max_new, max_kv=self.most,
                        scale=DIM ** -0.5, ctx=ctx, sync=False)
        self.free_count -= self.status[0]
        self.lens.copy_(self.kv_lens)
        return self.o(out.view(tokens, Q_HEADS * DIM), ctx)


def main() -> None:
    args = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    args.add_argument("--requests", type=int, default=8)
    args.add_argument("--prompt", type=int, default=141)
    args.add_argument("--steps", type=int, default=32)
    a = args.parse_args()
    ctx = hb.Context(torch.cuda.current_device())
    ctx.set_stream(torch.cuda.current_stream().cuda_stream)
    most = a.prompt + a.steps
    layer = Layer(a.requests, a.requests * -(-most // PAGE), most, ctx)
    gen = torch.Generator(device=DEV).manual_seed(1)
    lengths = [max(1, a.prompt - 3 * b) for b in range(a.requests)]
    x = torch.randn((sum(lengths), HIDDEN), generator=gen, device=DEV)
    layer.step(x, torch.tensor(lengths, dtype=torch.int32, device=DEV), max(lengths))
    one = _ints(a.requests, fill=1)
    x = torch.randn((a.requests, HIDDEN), generator=gen, device=DEV)
    torch.cuda.synchronize()
    start = time.perf_counter()
    for _ in range(a.steps):
        x = layer.step(x, one, 1)
        x = x / (x.norm(dim=-1, keepdim=True) / HIDDEN ** 0.5 + 1e-6)
    torch.cuda.synchronize()
    us = (time.perf_counter() - start) / a.steps * 1e6
    print(f"{a.requests} requests, prompts of {lengths[-1]} to {lengths[0]} tokens: "
          f"{us:.0f} us a step, lengths {layer.lens.tolist()}, "
          f"{int(layer.free_count)} pages free")


if __name__ == "__main__":
    main()
