"""The CPU stand-in for `crispybits_kernels._C` with attention operators added, for tests of host code only: a cache's values are
kept in a table beside its pages, quantised as the format defines."""
import torch

from oracle_backend import *  # noqa: F401,F403
from oracle_backend import IS_EMULATOR, fused_gate_up, fused_qkv, max_rho, packed_gemm, packed_gemv, sm_count, tile_n  # noqa: F401

_held = {}          # id of a cache -> {(page, offset): (k, v)} of all heads, and the cache itself (so that its id stays taken)


def kv4_block_bytes(head_dim, group_size):
    return 2 * 16 * (head_dim // 2 + 4 * (head_dim // group_size)) if head_dim % group_size == 0 else 0


def _quantised(x, group):
    g = x.double().unflatten(-1, (-1, group))
    lo = g.amin(-1, keepdim=True)
    scale = ((g.amax(-1, keepdim=True) - lo) / 15).to(x.dtype).double()
    code = torch.round((g - lo) / torch.where(scale == 0, torch.ones_like(scale), scale)).clamp(0, 15)
    return (torch.where(scale == 0, torch.zeros_like(code), code) * scale + lo).flatten(-2).to(x.dtype)


def _places(cache, table, starts, cu, n):
    if cu is None:
        per = n // table.shape[0]
        cu = torch.arange(table.shape[0] + 1) * per
    for s in range(table.shape[0]):
        for i in range(int(cu[s]), int(cu[s + 1])):
            p = int(starts[s]) + i - int(cu[s])
            yield i, s, (int(table[s, p // cache.page_size]), p % cache.page_size)


def kv4_append(cache, k, v, table, starts, cu):
    held = _held.setdefault(id(cache), ({}, cache))[0]
    k, v = _quantised(k, cache.group_size), _quantised(v, cache.group_size)
    for i, _, place in _places(cache, table, starts, cu, k.shape[0]):
        held[place] = (k[i], v[i])


def kv4_read(cache, table, starts, cu, n):
    held = _held[id(cache)][0]
    rows = [held[place] for _, _, place in _places(cache, table, starts, cu, n)]
    return torch.stack([r[0] for r in rows]), torch.stack([r[1] for r in rows])


def _attend(q, k, v, scale, hidden):
    share = q.shape[1] // k.shape[1]
    kk, vv = (x.double().repeat_interleave(share, 1).transpose(0, 1) for x in (k, v))
    s = (q.double().transpose(0, 1) @ kk.transpose(1, 2) * scale).masked_fill(hidden, float("-inf"))
    return (torch.softmax(s, -1).nan_to_num(0.0) @ vv).transpose(0, 1).to(q.dtype)


def kv4_attention(q, cache, table, lengths, scale):
    out = torch.zeros_like(q)
    q4, o4 = (x if q.dim() == 4 else x.unsqueeze(1) for x in (q, out))
    T = q4.shape[1]
    for b in range(q4.shape[0]):
        n = int(lengths[b])
        if n > 0:
            k, v = kv4_read(cache, table[b:b + 1], torch.zeros(1), torch.tensor([0, n]), n)
            o4[b] = _attend(q4[b], k, v, scale, torch.arange(n)[None] > torch.arange(T)[:, None] + n - T)
    return out


def prompt_attention(q, k, v, cu, cu_k, scale, causal, out=None):
    out = torch.zeros_like(q) if out is None else out
    for b in range(cu.numel() - 1):
        (a, e), (ka, ke) = (map(int, c[b:b + 2]) for c in (cu, cu_k))
        lq, lk = e - a, ke - ka
        hidden = torch.arange(lk)[None] > (torch.arange(lq)[:, None] + lk - lq if causal else lk)
        if lq and lk:
            out[a:e] = _attend(q[a:e], k[ka:ke], v[ka:ke], scale, hidden)
    return out
