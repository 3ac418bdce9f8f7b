"""Plain restatements of the training operators in 64 bits on the CPU: attention over a sorted edge list (reference ``graph_attention.py:237-273`` with
attention dropout and a length-bucket bias), EquivariantLayerNormV2 with what stands between two blocks (``equiformer/layer_norm.py:91-156``,
``gnn_block.py:164-218``) and channel dropout (``equiformer/drop.py:76-96``).  Forward passes only: gradients come from torch's autograd in 64 bits."""
from __future__ import annotations

import torch

from oracle import so3_oracle as so3

M32 = 0xFFFFFFFF


def philox(counter, key):
    """Philox4x32-10 on Python integers: 4 counter words, 2 key words -> 4 words"""
    c, k = list(counter), list(key)
    for _ in range(10):
        p0, p1 = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [(p1 >> 32) ^ c[1] ^ k[0], p1 & M32, (p0 >> 32) ^ c[3] ^ k[1], p0 & M32]
        k = [(k[0] + 0x9E3779B9) & M32, (k[1] + 0xBB67AE85) & M32]
    return c


def keep(rows: int, columns: int, first: int, p: float, seed: int, offset: int) -> torch.Tensor:
    """(rows, columns) factors 0 or 1 / (1 - p); column c of row r: word c % 4 of the counter (r, first + c // 4, offset)"""
    out = torch.zeros(rows, columns, dtype=torch.float64)
    threshold = int(p * 2.0 ** 32)
    for r in range(rows):
        for g in range((columns + 3) // 4):
            w = philox((r, first + g, offset & M32, (offset >> 32) & M32), (seed & M32, (seed >> 32) & M32))
            for i, x in enumerate(w):
                if 4 * g + i < columns and x >= threshold:
                    out[r, 4 * g + i] = 1.0 / (1.0 - p)
    return out


def act(x):
    return so3.C_SLRELU * (0.6 * x + 0.4 * x * (2.0 * torch.sigmoid(x) - 1.0))


def attention(alpha, value, alpha_dot, edge_dst, n_dst, edge_logits=None, edge_length=None, boundaries=None, table=None, mask=None):
    """64-bit tensors -> (n_dst, H, D); row by row"""
    E, H, _ = alpha.shape
    t = (act(alpha) * alpha_dot).sum(-1)
    if edge_logits is not None:
        dead = edge_logits == -float("inf")
        t = torch.where(dead[:, None], torch.full_like(t, -float("inf")), t + torch.where(dead, torch.zeros_like(edge_logits), edge_logits)[:, None])
    if table is not None:
        bucket = torch.zeros(E, dtype=torch.int64) if boundaries is None else (edge_length[:, None] >= boundaries[None, :]).sum(1)
        bias = table[bucket]
        t = torch.where(bias == -float("inf"), bias, t + torch.where(bias == -float("inf"), torch.zeros_like(bias), bias))
    rows = []
    for n in range(n_dst):
        at = (edge_dst == n).nonzero().flatten()
        tn, vn = t[at], value[at]
        live = tn != -float("inf")
        if len(at) == 0:
            rows.append(value.new_zeros(H, value.shape[2]))
            continue
        top = tn.detach().amax(0)
        top = torch.where(top == -float("inf"), torch.zeros_like(top), top)
        e = torch.where(live, torch.exp(torch.where(live, tn - top, torch.zeros_like(tn))), torch.zeros_like(tn))
        z = e.sum(0)
        p = e / torch.where(z == 0, torch.ones_like(z), z)
        if mask is not None:
            p = p * mask[at]
        rows.append(torch.where(p[..., None] == 0, torch.zeros_like(vn), p[..., None] * torch.where(p[..., None] == 0, torch.zeros_like(vn), vn)).sum(0))
    return torch.stack(rows) if rows else value.new_zeros(0, H, value.shape[2])


def per_channel(values, blocks):
    parts, at = [], 0
    for m, l in blocks:
        parts.append(values[:, at:at + m].repeat_interleave(2 * l + 1, 1))
        at += m
    return torch.cat(parts, 1)


def layer_norm(x, blocks, weight, bias, eps):
    parts, at, ch = [], 0, 0
    for m, l in blocks:
        d = 2 * l + 1
        f = x[:, at:at + m * d].reshape(-1, m, d)
        if l == 0:
            f = f - f.mean(1, keepdim=True)
        f = f * (f.pow(2).mean(-1).mean(1) + eps).pow(-0.5)[:, None, None] * weight[ch:ch + m][None, :, None]
        if l == 0:
            f = f + bias[None, :, None]
        parts.append(f.reshape(len(x), m * d))
        at, ch = at + m * d, ch + m
    return torch.cat(parts, 1)


def norm_gate_residual(x, y, blocks, scale=1.0, gate=None, post=None, mask=None, nxt=None, eps=1e-5):
    """post, nxt: (weight, bias) or None; mask: (rows, channels) factors"""
    h = x
    if y is not None:
        u = y if post is None else layer_norm(y, blocks, post[0], post[1], eps)
        if mask is not None:
            u = u * per_channel(mask, blocks)
        if gate is not None:
            u = u * per_channel(gate.repeat_interleave(len(x) // len(gate), 0), blocks)
        h = x + scale * u
    return h, (None if nxt is None else layer_norm(h, blocks, nxt[0], nxt[1], eps))
