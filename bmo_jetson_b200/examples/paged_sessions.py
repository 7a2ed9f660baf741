"""Batched sessions of a temporal transformer over a paged key-value cache.

The framework's batched frames keep one ring of n_ctx slots a session.  Here
the same layers (RMSNorm + QKV, RoPE, attention, O + residual, RMSNorm +
SwiGLU FFN + residual, on Q4_0 weights) run through the kernel layer with
the cache in pages: sessions of any length join, idle and end, and their pages go from one to
another.  One frame:

    book.plan                       block table and slot numbers of this frame's positions
    per layer:  bmo_k_batch_gemm_q4_0 (QKV, norm fused)
                cache.append        RoPE of q and k, fp16 or Q4_0 rows into their pages
                cache.attention     each session over its own window
                bmo_k_batch_gemm_q4_0 x 3 (O; FFN-in with norm and SwiGLU; FFN-out)

    python -m bmo_jetson_b200.examples.paged_sessions [--sessions 64 --frames 100 --kv q4_0 ...]

runs it on random weights and hidden states, with sessions ending and new ones
taking their place, and prints frames/s and the pages in use.
"""
from __future__ import annotations

import argparse
import time
from typing import List, Optional, Sequence

import numpy as np
import torch

from ..engine import KV_F16, KV_Q4_0, lib
from ..paged import PageBook, PagedKV

IDENTITY, SWIGLU = 0, 1
EPS = 1e-8


class Matrix:
    """A Q4_0 matrix in the row-tile layout and its batched product."""

    def __init__(self, blocks: torch.Tensor, rows: int, cols: int, swiglu_f: int = 0):
        """blocks: ggml Q4_0 rows as uint8 on the GPU."""
        self.rows, self.cols, self.f, self.perm = rows, cols, swiglu_f, SWIGLU if swiglu_f else IDENTITY
        n = lib().bmo_k_q4_0_tiled_bytes(rows, cols, self.perm, swiglu_f)
        self.tiles = torch.empty(n, dtype=torch.uint8, device=blocks.device)
        rc = lib().bmo_k_repack_q4_0(blocks.data_ptr(), self.tiles.data_ptr(), rows, cols, self.perm, swiglu_f,
                                     torch.cuda.current_stream().cuda_stream)
        if n == 0 or rc != 0:
            raise RuntimeError(f"bmo_k_repack_q4_0 rc={rc}")
        self.scratch = {}

    def __call__(self, x: torch.Tensor, gamma: Optional[torch.Tensor] = None,
                 resid: Optional[torch.Tensor] = None) -> torch.Tensor:
        n = x.shape[0]
        y = torch.empty((n, self.f or self.rows), device=x.device)
        if n not in self.scratch:
            size = lib().bmo_k_batch_gemm_scratch_bytes(self.rows, self.cols, self.perm, self.f, n)
            self.scratch[n] = torch.zeros(size, dtype=torch.uint8, device=x.device)
        s = self.scratch[n]
        rc = lib().bmo_k_batch_gemm_q4_0(self.tiles.data_ptr(), self.rows, self.cols, self.perm, self.f, x.data_ptr(),
                                         None if gamma is None else gamma.data_ptr(), EPS,
                                         None if resid is None else resid.data_ptr(), y.data_ptr(), n, 1, s.data_ptr(),
                                         s.numel(), torch.cuda.current_stream().cuda_stream)
        if rc != 0:
            raise RuntimeError(f"bmo_k_batch_gemm_q4_0 rc={rc}")
        return y


class Layer:
    def __init__(self, gamma1, qkv: Matrix, o: Matrix, gamma2, ffn_in: Matrix, ffn_out: Matrix):
        self.gamma1, self.qkv, self.o, self.gamma2, self.ffn_in, self.ffn_out = gamma1, qkv, o, gamma2, ffn_in, ffn_out


def random_blocks(rows: int, cols: int, gen: torch.Generator, sigma: float = 0.02) -> torch.Tensor:
    """Q4_0 blocks of about N(0, sigma) weights: random codes, one scale."""
    b = torch.randint(0, 256, (rows * cols // 32, 18), dtype=torch.uint8, device="cuda", generator=gen)
    scale = np.array([sigma / 4.6], np.float16).view(np.uint8)
    b[:, 0], b[:, 1] = int(scale[0]), int(scale[1])
    return b.reshape(-1)


def random_layers(n: int, dim: int, kv_dim: int, ffn: int, seed: int = 0) -> List[Layer]:
    gen = torch.Generator("cuda").manual_seed(seed)
    ones = torch.ones(dim, device="cuda")
    return [Layer(ones, Matrix(random_blocks(dim + 2 * kv_dim, dim, gen), dim + 2 * kv_dim, dim),
                  Matrix(random_blocks(dim, dim, gen), dim, dim), ones,
                  Matrix(random_blocks(2 * ffn, dim, gen), 2 * ffn, dim, ffn),
                  Matrix(random_blocks(dim, ffn, gen), dim, ffn)) for _ in range(n)]


class PagedSessions:
    """Up to n_req sessions of one stack of layers over a shared pool of pages."""

    def __init__(self, layers: Sequence[Layer], n_heads: int, n_kv_heads: int, head_dim: int, n_req: int, n_pages: int,
                 page_size: int = 16, max_len: int = 3000, window: int = 0, kv_type: int = KV_F16, theta: float = 10000.0):
        self.layers, self.n_heads, self.n_kv_heads, self.head_dim, self.theta = layers, n_heads, n_kv_heads, head_dim, theta
        self.book = PageBook.empty(n_req, n_pages, page_size, -(-max_len // page_size), window=window)
        self.cache = PagedKV.empty(self.book, len(layers), n_kv_heads, head_dim, kv_type)
        i32 = {"dtype": torch.int32, "device": self.book.device}
        self.lists = [torch.empty(n_req, **i32) for _ in range(3)]
        self.offsets = torch.empty(n_req + 1, **i32)
        self.status = torch.zeros(1, **i32)  # of all frames since it was looked at

    def frame(self, x: torch.Tensor, new: Sequence[int]) -> torch.Tensor:
        """One frame: new[r] 1 for a session that gets a position, 0 for an idle
        one, -1 for one that ends.  x [n, dim]: the hidden states of the n sessions
        that get a position, in order; returns theirs after the last layer, NaN if
        the frame was refused (refused() says why; the sessions are as before it)."""
        n = sum(1 for v in new if v > 0)
        if len(new) != self.book.lens.numel() or any(v > 1 for v in new):
            raise ValueError(f"new: 1, 0 or -1 for each of {self.book.lens.numel()} sessions")
        if x.shape[0] != n:
            raise ValueError(f"x: a row for each of the {n} sessions that get a position, got {x.shape[0]}")
        slot, pos, req = (t[:n] for t in self.lists)
        self.book.plan(torch.tensor(new, dtype=torch.int32).to(self.book.device, non_blocking=True), slot, pos, req,
                       self.offsets)
        self.status |= self.book.state[2]
        if n == 0:
            return x
        for i, layer in enumerate(self.layers):
            a = self.attend(i, layer.qkv(x, gamma=layer.gamma1), slot, pos, req)
            x = layer.o(a, resid=x)
            h = layer.ffn_in(x, gamma=layer.gamma2)
            x = layer.ffn_out(h, resid=x)
        return torch.where(self.book.state[2] == 0, x, torch.nan)  # without waiting for the plan

    def attend(self, i: int, qkv: torch.Tensor, slot: torch.Tensor, pos: torch.Tensor, req: torch.Tensor) -> torch.Tensor:
        """Layer i's attention of the projection's rows (q | k | v), which are rotated and stored on the way."""
        n, hd = qkv.shape[0], self.head_dim
        q_dim, kv_dim = self.n_heads * hd, self.n_kv_heads * hd
        q = qkv[:, :q_dim].unflatten(1, (self.n_heads, hd))
        k = qkv[:, q_dim:q_dim + kv_dim].unflatten(1, (self.n_kv_heads, hd))
        v = qkv[:, q_dim + kv_dim:].unflatten(1, (self.n_kv_heads, hd))
        self.cache.append(i, k, v, slot, pos=pos, q=q, q_out=q, theta=self.theta)
        a = torch.empty((n, q_dim), device=qkv.device)
        self.cache.attention(i, q, a.unflatten(1, (self.n_heads, hd)), rows=req)
        return a

    def refused(self) -> int:
        """Status bits of the plans since the last call of this (0: all frames were served); synchronises."""
        self.status |= self.book.state[2]
        bits = int(self.status)
        self.status.zero_()
        self.book.state[2] = 0
        return bits


def main(argv=None) -> int:
    ap = argparse.ArgumentParser(prog="python -m bmo_jetson_b200.examples.paged_sessions", description=__doc__.split("\n")[0])
    ap.add_argument("--sessions", type=int, default=64)
    ap.add_argument("--frames", type=int, default=100)
    ap.add_argument("--layers", type=int, default=32)
    ap.add_argument("--dim", type=int, default=4096)
    ap.add_argument("--heads", type=int, default=32)
    ap.add_argument("--kv-heads", type=int, default=32)
    ap.add_argument("--ffn", type=int, default=11264)
    ap.add_argument("--page-size", type=int, default=16)
    ap.add_argument("--window", type=int, default=512)
    ap.add_argument("--kv", choices=("f16", "q4_0"), default="q4_0")
    ap.add_argument("--seed", type=int, default=0)
    a = ap.parse_args(argv)
    if not 1 <= a.sessions <= 64 or a.dim % a.heads or a.dim // a.heads not in (64, 128) or a.heads % a.kv_heads:
        ap.error("1 to 64 sessions, heads of 64 or 128, a multiple of the key heads")
    hd = a.dim // a.heads
    longest = a.frames + 3
    pages = a.sessions * (-(-(a.window or longest) // a.page_size) + 2)
    s = PagedSessions(random_layers(a.layers, a.dim, a.kv_heads * hd, a.ffn, a.seed), a.heads, a.kv_heads, hd, a.sessions,
                      pages, a.page_size, longest, window=a.window, kv_type=KV_F16 if a.kv == "f16" else KV_Q4_0)
    rng = np.random.default_rng(a.seed)
    x = torch.randn(a.sessions, a.dim, device="cuda")
    rows, t0 = 0, 0.0
    for f in range(a.frames + 3):
        if f == 3:  # the first frames size scratch buffers
            torch.cuda.synchronize()
            t0, rows = time.perf_counter(), 0
        new = np.ones(a.sessions, int)
        gone = rng.random(a.sessions)
        new[gone < 0.01] = -1  # the session ends; its place takes a new one with the next frame
        new[(gone >= 0.01) & (gone < 0.03)] = 0
        n = int((new > 0).sum())
        y = s.frame(x[:n].contiguous(), new.tolist())
        rows += n
    torch.cuda.synchronize()
    dt = time.perf_counter() - t0
    refused = s.refused()
    print(f"{a.sessions} sessions, {a.layers} layers of {a.dim}, {a.kv} pages of {a.page_size}: {rows / dt:.0f} session "
          f"frames/s, {dt / a.frames * 1e3:.2f} ms a frame, {pages - int(s.book.state[1])} of {pages} pages in use, "
          f"status {refused}, finite {bool(torch.isfinite(y).all())}")
    return 0 if refused == 0 else 1


if __name__ == "__main__":
    raise SystemExit(main())
