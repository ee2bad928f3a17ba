"""The 4-bit key/value cache: append, read and attention against their definition in 64 bits.

    lo = min(x), scale = round_T((max(x) - lo) / 15), code = round_half_even((x - lo) / scale) <= 15, value = code * scale + lo
    out = softmax(scale * q K^T) V over the cached tokens that a row sees

What the bytes of a page mean is restated here (`Layout`), apart from the kernels' own arithmetic.
"""
import ctypes
import math

import pytest
import torch

DEV = "cuda"
FORMATS = [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128)]


# ------------------------------------------------------------------------------------------------ restatement
def quantise64(x, gs):
    """codes, scale, lo (double) of x [..., D], scale and lo as the cache's type holds them."""
    g = x.double().unflatten(-1, (-1, gs))
    lo = g.amin(-1)
    scale = ((g.amax(-1) - lo) / 15).to(x.dtype).double()
    safe = torch.where(scale == 0, torch.ones_like(scale), scale)
    codes = torch.round((g - lo[..., None]) / safe[..., None]).clamp(0, 15)
    return torch.where(scale[..., None] == 0, torch.zeros_like(codes), codes).flatten(-2), scale, lo


def values64(codes, scale, lo):
    gs = codes.shape[-1] // scale.shape[-1]
    return codes * scale.repeat_interleave(gs, -1) + lo.repeat_interleave(gs, -1)


class Layout:
    """Byte positions inside a page of one head: blocks of 16 tokens [K codes | K (scale, lo) | V codes | V (scale, lo)]."""

    def __init__(self, d, gs):
        self.d, self.gs, self.ng = d, gs, d // gs
        self.row, self.meta = d // 2, 4 * self.ng
        self.half = 16 * (self.row + self.meta)
        self.block = 2 * self.half

    def nibble(self, which, d, tok):
        """Number of the nibble, inside the 16 tokens' codes, of value d of token tok."""
        j, w = divmod(d, self.gs)
        lanes = 4 if which == "k" else 8              # lanes that share a token: each holds gs / lanes values of every group
        lane, i = divmod(w, self.gs // lanes)
        n = j * (self.gs // lanes) + i                # number of the value among the lane's
        if which == "k":
            return tok * self.d + lane * (self.d // 4) + n
        second = tok % 8 > 3                          # tokens t and 7 - t (and t + 8, 15 - t) share the bytes of two
        pair = (7 - tok % 8 if second else tok % 8) + 4 * (tok // 8)
        lane ^= 2 * (pair % 4) if self.d == 128 else 4 * (pair // 2 % 2)
        return pair * 2 * self.d + lane * (self.d // 4) + n // 4 * 8 + 4 * second + n % 4

    def put(self, page, which, off, codes, scale, lo, dtype):
        """Write one row (token `off` of the page) into page [bytes] (a CPU uint8 tensor)."""
        base = off // 16 * self.block + (self.half if which == "v" else 0)
        tok = off % 16
        for d in range(self.d):
            n = self.nibble(which, d, tok)
            at, shift = base + n // 2, 4 * (n % 2)
            page[at] = (int(page[at]) & ~(15 << shift) & 255) | int(codes[d]) << shift
        at = base + 16 * self.row + tok * self.meta
        pair = torch.stack((scale, lo), -1).to(dtype).contiguous().view(torch.uint8).flatten()
        page[at:at + self.meta] = pair


def test_layout_is_a_permutation_and_fills_a_block():
    from crispybits_kernels import _C
    for d, gs in FORMATS:
        lay = Layout(d, gs)
        for which in "kv":
            assert sorted(lay.nibble(which, i, tok) for i in range(d) for tok in range(16)) == list(range(16 * d))
        assert _C.kv4_block_bytes(d, gs) == lay.block and lay.block % 128 == 0
    for d, gs in ((64, 128), (96, 32), (128, 16), (0, 0), (256, 64), (128, 256)):
        assert _C.kv4_block_bytes(d, gs) == 0


# ------------------------------------------------------------------------------------------------ refusals, no GPU needed
def test_c_entry_points_refuse_bad_arguments():
    from crispybits_kernels import _C
    lib = _C._lib
    strides, s3 = (ctypes.c_int64 * 4)(8, 8, 8, 8), (ctypes.c_int64 * 3)(8, 8, 8)

    def cache(**kw):
        f = dict(pages=256, n_pages=4, kv_heads=2, head_dim=128, group_size=64, page_size=64, dtype=1)
        f.update(kw)
        return _C._KV4Cache(*(f[n] for n, _ in _C._KV4Cache._fields_))

    def append(c, k=256, v=256, st=strides, n=4, table=256, stride=2, seqs=2, starts=256, cu=256):
        return lib.cb_kv4_append(ctypes.byref(c) if c is not None else None, k, v, st, n, table, stride, seqs, starts, cu, 0)

    for bad in (dict(pages=0), dict(pages=8), dict(head_dim=96), dict(group_size=16), dict(head_dim=64, group_size=128),
                dict(page_size=24), dict(page_size=0), dict(dtype=0), dict(kv_heads=0), dict(n_pages=-1), dict(n_pages=1 << 31)):
        assert append(cache(**bad)) == 1 and lib.cb_last_error(), bad
    good = cache()
    assert append(None) == 1
    for bad in (dict(n=-1), dict(seqs=0), dict(n=5, cu=0), dict(k=0), dict(v=8), dict(starts=0), dict(table=0), dict(st=None),
                dict(st=(ctypes.c_int64 * 4)(8, 8, 4, 8)), dict(stride=-1)):
        assert append(good, **bad) == 1, bad
    assert append(good, n=0, k=0, v=0) == 0                    # nothing to do
    assert lib.cb_kv4_read(ctypes.byref(good), 0, 256, 4, 256, 2, 2, 256, 256, 0) == 1
    assert lib.cb_kv4_read(ctypes.byref(good), 256, 8, 4, 256, 2, 2, 256, 256, 0) == 1

    def attend(c=good, q=256, st=s3, out=256, B=2, T=1, H=4, table=256, stride=2, lengths=256, cnt=256, nc=1 << 20, part=256,
               np_=1 << 30):
        return lib.cb_kv4_attention(ctypes.byref(c), q, st, out, B, T, H, table, stride, lengths, 1.0, cnt, nc, part, np_, 0)

    for bad in (dict(H=3), dict(B=-1), dict(T=-1), dict(q=0), dict(out=4), dict(lengths=0), dict(st=None), dict(cnt=0), dict(nc=12),
                dict(st=(ctypes.c_int64 * 3)(8, 3, 8)), dict(part=0), dict(part=8), dict(c=cache(dtype=7)), dict(T=1 << 24)):
        assert attend(**bad) == 1, bad
    assert attend(B=0) == 0 and attend(T=0) == 0
    assert lib.cb_kv4_attention_counters(3, 4, 32, 8) == 3 * 8 and lib.cb_kv4_attention_counters(3, 5, 32, 8) == 3 * 8 * 2
    assert lib.cb_kv4_attention_counters(1, 1, 5, 2) == 0


def test_python_entry_points_refuse_cpu_tensors_and_bad_formats():
    import crispybits_kernels as ck
    for kw in (dict(head_dim=96), dict(head_dim=64, group_size=128), dict(head_dim=128, page_size=20), dict(head_dim=128, page_size=0),
               dict(head_dim=128, dtype=torch.float32)):
        with pytest.raises(ValueError):
            ck.KV4Cache.empty(2, 2, device="cpu", **kw)
    with pytest.raises(ValueError):
        ck.KV4Cache.empty(0, 2, 64, device="cpu")
    c = ck.KV4Cache.empty(2, 2, 64, device="cpu")
    assert (c.n_pages, c.kv_heads, c.pages.shape[2]) == (2, 2, 4 * Layout(64, 64).block)
    i32 = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError):
        ck.kv4_append(c, torch.zeros(1, 2, 64).half(), torch.zeros(1, 2, 64).half(), i32[None], i32)
    with pytest.raises(RuntimeError):
        ck.kv4_attention(torch.zeros(1, 2, 64).half(), c, i32[None], i32)
    with pytest.raises(RuntimeError):
        ck.kv4_read(c, i32[None], i32, None, 1)


def test_python_struct_mirror_matches_the_c_header(tmp_path):
    import os
    import subprocess

    from conftest import ROOT
    from crispybits_kernels import _C
    lines = ['printf("%zu\\n", sizeof(cb_kv4_cache));'] + [f'printf("%zu\\n", offsetof(cb_kv4_cache, {f}));' for f, _ in _C._KV4Cache._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "crispybits_b200.h"\nint main(void) {\n' + "\n".join(lines) + "\nreturn 0; }\n")
    subprocess.run(["gcc", "-std=c99", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "layout")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [ctypes.sizeof(_C._KV4Cache)] + [getattr(_C._KV4Cache, f).offset for f, _ in _C._KV4Cache._fields_]


# ------------------------------------------------------------------------------------------------ GPU: append and read
def i32(values, device=DEV):
    return torch.tensor(values, dtype=torch.int32, device=device)


def rand_kv(n, heads, d, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, heads, d, generator=g) * (0.5 + 3.0 * (torch.rand(heads, d, generator=g) > 0.95))
    return x.to(dtype).to(DEV)


def table_for(need, n_pages, seed):
    """Rows of distinct pages in random order; the rest of each row holds page numbers that do not exist."""
    ids = torch.randperm(n_pages, generator=torch.Generator().manual_seed(seed)).tolist()
    rows, at = [], 0
    for n in need:
        rows.append(ids[at:at + n] + [-1] * (max(need) - n))
        at += n
    return rows


def offsets(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d,gs", FORMATS)
@pytest.mark.parametrize("page", [16, 48, 64])
def test_append_writes_exactly_the_defined_bytes(dtype, d, gs, page):
    """Every byte of the pool: the rows of the new tokens as defined, everything else as it was."""
    import crispybits_kernels as ck
    heads, lens, starts = 3, [1, 17, 0, 70, 5], [0, 15, 9, 31, 63]
    need = [max(1, -(-(s + n) // page)) for s, n in zip(starts, lens)]
    cache = ck.KV4Cache.empty(sum(need) + 1, heads, d, page, gs, dtype, DEV)
    pool = torch.randint(0, 256, cache.pages.shape, generator=torch.Generator().manual_seed(7), dtype=torch.uint8)
    cache.pages.copy_(pool)
    rows = table_for(need, sum(need) + 1, 3)
    k, v = rand_kv(sum(lens), heads, d, dtype, 1), rand_kv(sum(lens), heads, d, dtype, 2)
    ck.kv4_append(cache, k, v, i32(rows), i32(starts), i32(offsets(lens)))
    lay = Layout(d, gs)
    for name, x in (("k", k), ("v", v)):
        codes, scale, lo = (t.cpu() for t in quantise64(x, gs))
        i = 0
        for s, n in enumerate(lens):
            for p in range(starts[s], starts[s] + n):
                for h in range(heads):
                    lay.put(pool[rows[s][p // page], h], name, p % page, codes[i, h], scale[i, h], lo[i, h], dtype)
                i += 1
    got = cache.pages.cpu()
    assert torch.equal(got, pool), f"{int((got != pool).sum())} bytes differ"
    # and back: one rounding of code * scale + lo in fp32 (2^-24 of its larger part), one to the type
    gk, gv = ck.kv4_read(cache, i32(rows), i32(starts), i32(offsets(lens)), sum(lens))
    for got_x, x in ((gk, k), (gv, v)):
        codes, scale, lo = quantise64(x, gs)
        want = values64(codes, scale, lo)
        size = (15 * scale + lo.abs()).repeat_interleave(gs, -1)
        tol = torch.finfo(dtype).eps / 2 * want.abs() * (1 + 2 ** -20) + 2.0 ** -24 * size + 2.0 ** -25
        assert ((got_x.double() - want).abs() <= tol).all()
        # each value is within half a step of what was appended (and the rounding of scale: 15 eps / 2 of a step)
        step = scale.repeat_interleave(gs, -1)
        assert ((want - x.double()).abs() <= step * (0.5 + 15 * torch.finfo(dtype).eps)).all()


@pytest.mark.gpu
def test_append_forms_and_strides_agree():
    """[B, H, D], [B, T, H, D], packed, column slices of a fused projection and misaligned rows: the same bytes."""
    import crispybits_kernels as ck
    B, T, heads, d = 3, 4, 2, 64
    fused = rand_kv(B * T, 3 * heads + 1, d, torch.float16, 5).flatten(1)
    k, v = fused[:, heads * d:2 * heads * d].view(-1, heads, d), fused[:, 2 * heads * d:3 * heads * d].view(-1, heads, d)
    odd = torch.empty(k.numel() + 1, dtype=torch.float16, device=DEV)[1:].view(k.shape).copy_(k)
    assert odd.data_ptr() % 16 and not k.is_contiguous()
    rows, starts = i32(table_for([1] * B, B, 1)), i32([3, 0, 60 - T])

    def bytes_of(*args):
        c = ck.KV4Cache.empty(B, heads, d)
        c.pages.zero_()
        ck.kv4_append(c, *args)
        return c.pages

    want = bytes_of(k.contiguous(), v.contiguous(), rows, starts, i32([0, T, 2 * T, 3 * T]))
    assert want.any()
    assert torch.equal(want, bytes_of(k, v, rows, starts, i32([0, T, 2 * T, 3 * T])))
    assert torch.equal(want, bytes_of(odd, v, rows, starts))
    assert torch.equal(want, bytes_of(k.view(B, T, heads, d), v.reshape(B, T, heads, d), rows, starts))
    heads_first = k.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(want, bytes_of(heads_first, v, rows, starts))
    # token by token, as decode steps do
    c = ck.KV4Cache.empty(B, heads, d)
    c.pages.zero_()
    for j in range(T):
        ck.kv4_append(c, k.view(B, T, heads, d)[:, j], v.view(B, T, heads, d)[:, j], rows, starts + j)
    assert torch.equal(want, c.pages)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_append_edge_values(dtype):
    """Constant groups, zeros, negative zero, ties, the type's largest values, subnormal ranges, infinities and NaN."""
    import crispybits_kernels as ck
    d, gs, big = 64, 32, torch.finfo(dtype).max
    if dtype == torch.bfloat16:
        big = 2.0 ** 126            # the range of a group has to be a float
    rows = [torch.full((d,), 3.0), torch.zeros(d), torch.linspace(-1, 1, d), torch.arange(d) * 0.5 - 7.5,
            torch.cat((torch.full((16,), -big), torch.full((48,), big))), torch.full((d,), -big),
            torch.arange(d) * torch.finfo(dtype).tiny / 64, torch.arange(d) % 16 * 1.0, torch.arange(d) % 31 * 0.5,
            torch.cat((torch.full((31,), 1.0), torch.full((33,), 1.0 + torch.finfo(dtype).eps)))]
    x = torch.stack(rows).to(dtype).to(DEV)[:, None]                     # [n, 1, d]
    n = x.shape[0]
    c = ck.KV4Cache.empty(1, 1, d, 64, gs, dtype)
    ck.kv4_append(c, x, -x, i32([[0]]), i32([0]), i32([0, n]))
    gk, gv = ck.kv4_read(c, i32([[0]]), i32([0]), i32([0, n]), n)
    for got, src in ((gk, x), (gv, -x)):
        codes, scale, lo = quantise64(src, gs)
        if dtype == torch.bfloat16:
            small = scale < 2.0 ** -126
            scale = torch.where(small, 0.0, scale)
            codes = torch.where(small.repeat_interleave(gs, -1), 0.0, codes)
        # scale is rounded: 65504 of a range of 131008 stands for 15 * 8736 - 65504 = 65536, which fp16 does not have
        want = values64(codes, scale, lo).clamp(-torch.finfo(dtype).max, torch.finfo(dtype).max)
        size = (15 * scale + lo.abs()).repeat_interleave(gs, -1)
        tol = torch.finfo(dtype).eps / 2 * want.abs() * (1 + 2 ** -20) + 2.0 ** -24 * size + torch.finfo(dtype).tiny * torch.finfo(dtype).eps
        over = ((got.double() - want).abs() - tol).amax(-1).flatten().tolist()
        assert max(over) <= 0, over
    y = x.clone()
    y[2, 0, 5], y[3, 0, 40], y[7, 0, 0] = math.nan, math.inf, -math.inf
    ck.kv4_append(c, y, y, i32([[0]]), i32([0]), i32([0, n]))
    gk, gv = ck.kv4_read(c, i32([[0]]), i32([0]), i32([0, n]), n)
    bad = torch.zeros(n, 1, d, dtype=torch.bool, device=DEV)
    bad[2, 0, :32] = bad[3, 0, 32:] = bad[7, 0, :32] = True
    assert torch.equal(gk.isnan(), bad) and torch.equal(gv.isnan(), bad)


@pytest.mark.gpu
def test_tokens_without_a_place_are_left_out():
    import crispybits_kernels as ck
    from crispybits_kernels import _C
    d, heads, page = 64, 2, 16
    k, v = rand_kv(40, heads, d, torch.float16, 1), rand_kv(40, heads, d, torch.float16, 2)
    _C.decode_status()
    # sequence 0: its second page does not exist (-1, then one past the end); sequence 1 runs over the table's end; starts below 0
    for wrong in (-1, 3, -(1 << 31), (1 << 31) - 1):
        c = ck.KV4Cache.empty(3, heads, d, page)
        c.pages.fill_(0xAB)
        table = i32([[0, wrong], [1, 2]])
        ck.kv4_append(c, k, v, table, i32([10, 25]), i32([0, 20, 40]))
        assert _C.decode_status() == 3001 and _C.decode_status() == 0
        good = ck.KV4Cache.empty(3, heads, d, page)
        good.pages.fill_(0xAB)
        ck.kv4_append(good, torch.cat((k[:6], k[20:27])), torch.cat((v[:6], v[20:27])), i32([[0, 0], [1, 2]]), i32([10, 25]), i32([0, 6, 13]))
        assert torch.equal(c.pages, good.pages) and _C.decode_status() == 0
        gk, _ = ck.kv4_read(c, table, i32([10, 25]), i32([0, 20, 40]), 40)
        assert torch.equal(gk[:6], ck.kv4_read(good, i32([[0, 0], [1, 2]]), i32([10, 25]), i32([0, 6, 13]), 13)[0][:6])
        assert _C.decode_status() == 3001
    c.pages.fill_(0xAB)
    ck.kv4_append(c, k, v, i32([[0, 1]]), i32([-50]), i32([0, 40]))
    assert (c.pages == 0xAB).all() and _C.decode_status() == 3001
    # tokens before the first and behind the last sequence belong to none: no error
    ck.kv4_append(c, k, v, i32([[0, 1]]), i32([0]), i32([3, 5]))
    assert _C.decode_status() == 0
    gk, _ = ck.kv4_read(c, i32([[0, 1]]), i32([0]), i32([0, 2]), 2)
    codes, scale, lo = quantise64(k[3:5], 64)
    assert (gk.double() - values64(codes, scale, lo)).abs().max() < 2e-2
    assert (c.pages[2] == 0xAB).all()


# ------------------------------------------------------------------------------------------------ GPU: attention
class Filled:
    """A cache with sequences of the given lengths, and the values it holds in 64 bits."""

    def __init__(self, lens, heads, d, gs, page, dtype, seed=0, spare=2, k_gain=1.0):
        import crispybits_kernels as ck
        need = [max(1, -(-n // page)) for n in lens]
        self.lens, self.rows = lens, table_for(need, sum(need) + spare, seed + 3)
        self.cache = ck.KV4Cache.empty(sum(need) + spare, heads, d, page, gs, dtype)
        self.cache.pages.fill_(0xFF)                       # what was never appended: NaN scales, codes 15
        self.k, self.v = rand_kv(sum(lens), heads, d, dtype, seed) * k_gain, rand_kv(sum(lens), heads, d, dtype, seed + 1)
        self.table, self.lengths = i32(self.rows), i32(lens)
        ck.kv4_append(self.cache, self.k, self.v, self.table, i32([0] * len(lens)), i32(offsets(lens)))
        self.gs = gs

    def reference(self, q, scale=None, drop=None):
        """(out, tolerance) for q [B, T, H, D]; drop[b]: positions left out.

        Tolerance, for each output: the final rounding; the weights' rounding to fp16; the scores' error -- fp32 sums of 2 D products, and
        of D code products each cut to the accumulator's width, 2^-20 of their absolute sum is ample -- which moves every weight
        and their sum by exp of it.
        The weights' rounding: with x = p s (s the group's scale) and w = fp16(x), |w - x| <= 2^-11 x, the kernel forms
        sum w code + sum (p (lo + 7.5 s) - 7.5 w) = sum p (code s + lo) + sum (w - x) (code - 7.5), so 2^-11 sum p s |code - 7.5|; its fp32 sums of
        terms as large as 7.5 p s, which cancel, are off by 2^-20 of those at most."""
        B, T, H, D = q.shape
        scale = D ** -0.5 if scale is None else scale
        heads = self.cache.kv_heads
        out, tol = torch.zeros(B, T, H, D, dtype=torch.double, device=DEV), torch.zeros(B, T, H, D, dtype=torch.double, device=DEV)
        parts = [quantise64(x, self.gs) for x in (self.k, self.v)]
        at = offsets(self.lens)
        for b, n in enumerate(self.lens):
            (kc, ks, kl), (vc, vs, vl) = ([t[at[b]:at[b + 1]] for t in part] for part in parts)
            kv, vv = values64(kc, ks, kl), values64(vc, vs, vl)
            vcode = values64(vc, vs, torch.zeros_like(vl))
            vhalf = 7.5 * values64(torch.ones_like(vc), vs, torch.zeros_like(vl))
            kabs = values64(kc, ks, kl.abs())
            pos = torch.arange(n, device=DEV)
            for j in range(T):
                seen = pos < n - T + 1 + j
                if drop is not None:
                    for p in drop[b]:
                        seen &= pos != p
                if not seen.any():
                    continue
                for h in range(H):
                    g = h // (H // heads)
                    qq = q[b, j, h].double()
                    w = torch.softmax((kv[seen, g] @ qq) * scale, 0)
                    err = 2.0 ** -20 * ((kabs[seen, g] @ qq.abs()) * abs(scale)).max()
                    out[b, j, h] = w @ vv[seen, g]
                    tol[b, j, h] = (torch.finfo(q.dtype).eps / 2 * out[b, j, h].abs() * 1.01 + 2.0 ** -11 * 1.01 * (w @ (vcode - vhalf)[seen, g].abs())
                                    + 2.0 ** -20 * (w @ vhalf[seen, g])
                                    + 2 * (err + 2.0 ** -21) * (w @ (vcode[seen, g] + vl.abs().repeat_interleave(self.gs, -1)[seen, g])) + 1e-7)
        return out, tol


def check(got, want):
    out, tol = want
    over = (got.double() - out).abs() - tol
    assert torch.isfinite(got).all() and (over <= 0).all(), f"{over.max():.2e} over, at tolerance {tol[over == over.max()][0]:.2e}"


def rand_q(B, T, H, D, dtype, seed=9):
    return torch.randn(B, T, H, D, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d,gs", FORMATS)
@pytest.mark.parametrize("T,group,page", [(1, 1, 64), (1, 8, 16), (3, 4, 32), (5, 2, 80)])
def test_attention_matches_the_definition(dtype, d, gs, T, group, page):
    import crispybits_kernels as ck
    heads, lens = 3, [1, 0, 2, 15, 16, 17, 333, 64, 700]
    f = Filled(lens, heads, d, gs, page, dtype, seed=d + gs)
    q = rand_q(len(lens), T, heads * group, d, dtype)
    got = ck.kv4_attention(q, f.cache, f.table, f.lengths)
    check(got, f.reference(q))
    for b, n in enumerate(lens):
        for j in range(T):
            if n - T + 1 + j <= 0:
                assert (got[b, j] == 0).all()
    if T == 1:
        assert torch.equal(got[:, 0], ck.kv4_attention(q[:, 0], f.cache, f.table, f.lengths))


@pytest.mark.gpu
@pytest.mark.parametrize("B,heads,group,n", [(1, 1, 1, 1), (1, 1, 1, 5000), (1, 2, 16, 2500), (2, 1, 71, 400), (40, 5, 1, 33), (300, 1, 2, 20)])
def test_attention_over_shapes(B, heads, group, n):
    """One head and one long sequence, many query heads, many short sequences (more of them than a warp scans at once)."""
    import crispybits_kernels as ck
    lens = [max(0, n - 7 * (b % 4)) for b in range(B)]
    f = Filled(lens, heads, 64, 32, 32, torch.float16, seed=n)
    q = rand_q(B, 1, heads * group, 64, torch.float16)
    check(ck.kv4_attention(q, f.cache, f.table, f.lengths), f.reference(q))


@pytest.mark.gpu
def test_attention_scale_strides_and_sharp_scores():
    import crispybits_kernels as ck
    f = Filled([200, 77], 2, 128, 128, 64, torch.bfloat16, k_gain=8.0)
    wide = rand_q(2, 2, 11, 128, torch.bfloat16) * 4
    q = wide[:, :, 3:7]                                            # a slice of a fused projection
    want = f.reference(q, 0.5)
    got = ck.kv4_attention(q, f.cache, f.table, f.lengths, scale=0.5)
    check(got, want)
    assert torch.equal(got, ck.kv4_attention(q.contiguous(), f.cache, f.table, f.lengths, 0.5))
    odd = torch.empty(q.numel() + 1, dtype=q.dtype, device=DEV)[1:].view(q.shape).copy_(q)
    assert torch.equal(got, ck.kv4_attention(odd, f.cache, f.table, f.lengths, 0.5))
    t = q.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(got, ck.kv4_attention(t, f.cache, f.table, f.lengths, 0.5))


@pytest.mark.gpu
def test_attention_value_scales_of_very_different_size():
    """Values of most tokens 2^-9 of a few tokens': the weights are rounded against the largest scale met."""
    import crispybits_kernels as ck
    f = Filled([600], 1, 64, 32, 16, torch.float16)
    f.v[::3] *= 2.0 ** -9
    f.v[5] *= 64.0
    ck.kv4_append(f.cache, f.k, f.v, f.table, i32([0]), i32([0, 600]))
    q = rand_q(1, 2, 4, 64, torch.float16)
    check(ck.kv4_attention(q, f.cache, f.table, f.lengths), f.reference(q))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n", [2, 33, 700])
def test_attention_groups_with_one_large_value(dtype, n):
    """Most codes of a group are then at one end."""
    import crispybits_kernels as ck
    f = Filled([n], 2, 128, 64, 64, dtype)
    f.v[..., 7::64] = f.v[..., 7::64].abs() * 100
    f.v[..., 64:] *= -1
    ck.kv4_append(f.cache, f.k, f.v, f.table, i32([0]), i32([0, n]))
    q = rand_q(1, 2, 8, 128, dtype)
    check(ck.kv4_attention(q, f.cache, f.table, f.lengths), f.reference(q))


@pytest.mark.gpu
def test_attention_ignores_what_a_row_does_not_see():
    """Infinities and NaN in tokens behind the length, and in the newest token for the rows before it."""
    import crispybits_kernels as ck
    f = Filled([100, 50], 2, 128, 64, 64, torch.float16)
    q = rand_q(2, 3, 4, 128, torch.float16)
    want = ck.kv4_attention(q, f.cache, f.table, f.lengths)
    bad = torch.full((2, 2, 128), math.nan, dtype=torch.float16, device=DEV)
    bad[1] = math.inf
    ck.kv4_append(f.cache, bad, bad, f.table, f.lengths)           # one token more, not counted by lengths
    assert torch.equal(want, ck.kv4_attention(q, f.cache, f.table, f.lengths))
    got = ck.kv4_attention(q, f.cache, f.table, f.lengths + 1)     # now the last row of each sequence sees it
    assert got[:, 2].isnan().all() and torch.isfinite(got[:, :2]).all()
    # rows 0 and 1 see what rows 1 and 2 saw before
    out, tol = f.reference(torch.cat((q[:, :1], q[:, :2]), 1))
    check(got[:, :2], (out[:, 1:], tol[:, 1:]))


@pytest.mark.gpu
def test_attention_leaves_out_pages_that_do_not_exist():
    import crispybits_kernels as ck
    from crispybits_kernels import _C
    f = Filled([100, 90], 1, 64, 64, 16, torch.float16)
    q = rand_q(2, 1, 2, 64, torch.float16)
    _C.decode_status()
    table = f.table.clone()
    table[0, 2], table[1, 0], table[1, 5] = -1, f.cache.n_pages, (1 << 31) - 1
    got = ck.kv4_attention(q, f.cache, table, f.lengths)
    assert _C.decode_status() == 3001 and _C.decode_status() == 0
    check(got, f.reference(q, drop=[range(32, 48), [*range(16), *range(80, 96)]]))
    none = torch.full_like(table, -5)
    assert (ck.kv4_attention(q, f.cache, none, f.lengths) == 0).all() and _C.decode_status() == 3001
    # lengths below zero see nothing, beyond the table everything there is (all six pages full)
    full = Filled([96, 96], 1, 64, 64, 16, torch.float16)
    got = ck.kv4_attention(q, full.cache, full.table, i32([-3, 1 << 30]))
    assert (got[0] == 0).all() and torch.equal(got[1], ck.kv4_attention(q, full.cache, full.table, full.lengths)[1])
    assert torch.isfinite(got).all() and _C.decode_status() == 0


@pytest.mark.gpu
def test_attention_is_the_same_every_time_on_any_stream_and_captured():
    import crispybits_kernels as ck
    f = Filled([3000, 10, 1500], 2, 128, 64, 64, torch.bfloat16)
    q = rand_q(3, 1, 8, 128, torch.bfloat16)
    want = ck.kv4_attention(q, f.cache, f.table, f.lengths)
    check(want, f.reference(q))
    for _ in range(5):
        assert torch.equal(want, ck.kv4_attention(q, f.cache, f.table, f.lengths))
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(3)], []
    for s in streams * 4:
        with torch.cuda.stream(s):
            outs.append(ck.kv4_attention(q, f.cache, f.table, f.lengths))
    torch.cuda.synchronize()
    assert all(torch.equal(want, o) for o in outs)
    graphs = []
    for _ in range(2):                                             # two graphs that run at the same time
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = [ck.kv4_attention(q, f.cache, f.table, f.lengths) for _ in range(3)]
        graphs.append((g, outs))
    for _ in range(10):
        for (g, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(want, o) for _, outs in graphs for o in outs)
    # a replay reads what the index tensors hold then
    f.lengths.copy_(i32([2999, 0, 1]))
    graphs[0][0].replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][1][0], ck.kv4_attention(q, f.cache, f.table, f.lengths)) and (graphs[0][1][0][1] == 0).all()


@pytest.mark.gpu
def test_a_captured_decode_step_appends_and_attends():
    """One step's append and attention captured, replayed for several tokens: as eager steps."""
    import crispybits_kernels as ck
    B, heads, d, steps, dt = 3, 2, 64, 20, torch.float16
    k, v = rand_kv(B * steps, heads, d, dt, 1).view(steps, B, heads, d), rand_kv(B * steps, heads, d, dt, 2).view(steps, B, heads, d)
    q = torch.stack([rand_q(B, 1, 4, d, dt, s)[:, 0] for s in range(steps)])
    table = i32(table_for([2] * B, 2 * B, 4))

    def fresh():
        c = ck.KV4Cache.empty(2 * B, heads, d, 16)
        return c, i32([0, 3, 11])

    c, n = fresh()
    ck.kv4_append(c, v[0].repeat(11, 1, 1)[:14], k[0].repeat(11, 1, 1)[:14], table, i32([0, 0, 0]), i32([0, 0, 3, 14]))
    start = c.pages.clone()
    eager = []
    for s in range(steps):
        ck.kv4_append(c, k[s], v[s], table, n)
        n = n + 1
        eager.append(ck.kv4_attention(q[s], c, table, n))
    pages = c.pages.clone()
    c.pages.copy_(start)
    n = i32([0, 3, 11])
    sk, sv, sq = k[0].clone(), v[0].clone(), q[0].clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ck.kv4_append(c, sk, sv, table, n)
        n += 1
        out = ck.kv4_attention(sq, c, table, n)
    for s in range(steps):
        sk.copy_(k[s]); sv.copy_(v[s]); sq.copy_(q[s])
        g.replay()
        assert torch.equal(out, eager[s]), s
    assert torch.equal(c.pages, pages)


@pytest.mark.gpu
def test_pages_beyond_32_bit_offsets():
    import crispybits_kernels as ck
    heads, d, page = 64, 128, 64
    per_page = heads * 4 * Layout(d, 64).block
    n_pages = (1 << 32) // per_page + 40
    c = ck.KV4Cache.empty(n_pages, heads, d, page)
    lens = [130, 64]
    table = i32([[n_pages - 1, n_pages - 20, 7], [n_pages - 3, 0, 0]])
    k, v = rand_kv(194, heads, d, torch.float16, 1), rand_kv(194, heads, d, torch.float16, 2)
    small = ck.KV4Cache.empty(5, heads, d, page)
    table_small = i32([[0, 1, 2], [3, 0, 0]])
    q = rand_q(2, 1, heads, d, torch.float16)
    res = []
    for cache, tab in ((c, table), (small, table_small)):
        ck.kv4_append(cache, k, v, tab, i32([0, 0]), i32([0, 130, 194]))
        res.append((*ck.kv4_read(cache, tab, i32([0, 0]), i32([0, 130, 194]), 194), ck.kv4_attention(q, cache, tab, i32(lens))))
    for a, b in zip(*res):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_a_cache_can_be_copied_and_pickled():
    import copy
    import dataclasses
    import io

    import crispybits_kernels as ck
    f = Filled([40], 1, 64, 32, 16, torch.float16)
    q = rand_q(1, 1, 2, 64, torch.float16)
    want = ck.kv4_attention(q, f.cache, f.table, f.lengths)
    buf = io.BytesIO()
    torch.save(f.cache, buf)
    buf.seek(0)
    moved = dataclasses.replace(f.cache, pages=f.cache.pages.clone())
    for other in (copy.deepcopy(f.cache), torch.load(buf, weights_only=False), moved):
        assert other.pages.data_ptr() != f.cache.pages.data_ptr()
        assert torch.equal(want, ck.kv4_attention(q, other, f.table, f.lengths))
        other.pages.zero_()
        assert torch.equal(want, ck.kv4_attention(q, f.cache, f.table, f.lengths))


@pytest.mark.gpu
def test_captures_beyond_the_prepared_counters():
    """Counters cut from the slab are never given out twice; when it is used up, a graph zeroes its own."""
    import crispybits_kernels as ck
    from crispybits_kernels import _C
    f = Filled([2000, 30], 2, 64, 64, 64, torch.float16)
    q = rand_q(2, 1, 4, 64, torch.float16)
    want = ck.kv4_attention(q, f.cache, f.table, f.lengths)
    slab = _C._attention_slab[torch.cuda.current_device()]
    before = slab[1]
    slab[1] = slab[0].numel() - 40                                 # room for one call more
    try:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = [ck.kv4_attention(q, f.cache, f.table, f.lengths) for _ in range(3)]
        for _ in range(3):
            g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(want, o) for o in outs) and slab[1] == slab[0].numel() - 8
    finally:
        slab[1] = before


@pytest.mark.gpu
def test_shapes_and_devices_that_do_not_fit_are_refused():
    import crispybits_kernels as ck
    f = Filled([20], 2, 64, 32, 16, torch.float16)
    q = rand_q(1, 1, 4, 64, torch.float16)
    k = f.k[:1]
    ok = (f.table, f.lengths)
    for args in ((q.bfloat16(), f.cache, *ok), (q[..., :32], f.cache, *ok), (q[:, :, :3], f.cache, *ok), (q.cpu(), f.cache, *ok),
                 (q, f.cache, f.table.long(), f.lengths), (q, f.cache, f.table, f.lengths.long()), (q, f.cache, f.table.cpu(), f.lengths),
                 (q, f.cache, f.table, i32([1, 2])), (q.repeat(2, 1, 1, 1), f.cache, *ok), (q, f.cache, f.table[0], f.lengths),
                 (q, f.cache, f.table.repeat(1, 2)[:, ::2], f.lengths)):
        with pytest.raises(RuntimeError):
            ck.kv4_attention(*args)
    for args in ((k.float(), k, *ok), (k, k[:, :1], *ok), (k[..., :32], k[..., :32], *ok), (k, k.cpu(), *ok),
                 (k, k, f.table, f.lengths.cpu()), (k, k, *ok, i32([0, 1, 1])), (k, k, *ok, torch.tensor([0, 1], device=DEV))):
        with pytest.raises(RuntimeError):
            ck.kv4_append(f.cache, *args)
    with pytest.raises(ValueError):
        ck.kv4_append(f.cache, f.k[:3], f.k[:3], f.table.repeat(2, 1), i32([0, 0]))
    with pytest.raises(RuntimeError):
        ck.kv4_read(f.cache, *ok, None, -1)
    wrong = ck.KV4Cache(f.cache.pages, 128, 16, 32, torch.float16)
    with pytest.raises(RuntimeError):
        ck.kv4_attention(rand_q(1, 1, 4, 128, torch.float16), wrong, *ok)
    assert ck.kv4_attention(q[:, :0], f.cache, *ok).shape == (1, 0, 4, 64)
    ck.kv4_append(f.cache, k[:0], k[:0], *ok, i32([0, 0]))


# ------------------------------------------------------------------------------------------------ GPU: values that are not finite
def check_with_nan(got, want):
    """NaN exactly where the definition has NaN, everything else within its tolerance."""
    out, tol = want
    assert torch.equal(got.isnan(), out.isnan()), f"{int((got.isnan() != out.isnan()).sum())} of {got.numel()} values"
    there = ~out.isnan()
    assert ((got.double() - out).abs() <= tol)[there].all() and torch.isfinite(got[there]).all()


# One path through the work each: parts of long sequences, whole segments and parts of several CTAs, segments of single warps, the last two mixed.
NON_FINITE_SHAPES = [([2500, 1, 700, 16], 2), ([900, 333, 1, 64, 5, 700] * 3, 4), ([20, 1, 128, 50] * 19, 2), ([100, 1, 129, 600] * 10, 4)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens,heads", NON_FINITE_SHAPES)
@pytest.mark.parametrize("T,group", [(1, 1), (2, 8)])
def test_queries_that_are_not_finite_give_nan_on_every_path(dtype, lens, heads, T, group):
    """A NaN or an infinity among a query's values makes each of its scores NaN or infinite, none of which a softmax survives: its row is NaN,
    unless it sees nothing, and the rows beside it are untouched."""
    import crispybits_kernels as ck
    f = Filled(lens, heads, 64, 32, 32, dtype)
    q = rand_q(len(lens), T, heads * group, 64, dtype)
    want = f.reference(q)
    rows = torch.zeros(q.shape[:3], dtype=torch.bool, device=DEV)
    for i, (b, h) in enumerate((b, h) for b in range(len(lens)) for h in (0, heads * group - 1)):
        q[b, T - 1, h, (7 * i) % 64] = (math.nan, math.inf, -math.inf)[i % 3]
        rows[b, T - 1, h] = True
    out = torch.where(rows[..., None] & (f.lengths > 0)[:, None, None, None], math.nan, want[0])
    check_with_nan(ck.kv4_attention(q, f.cache, f.table, f.lengths), (out, want[1]))


@pytest.mark.gpu
@pytest.mark.parametrize("lens,heads", NON_FINITE_SHAPES)
def test_keys_that_are_not_finite_give_nan_on_every_path(lens, heads):
    """One token, a block, hundreds of tokens or a whole sequence of keys with a NaN or an infinity: every row that sees one is NaN."""
    import crispybits_kernels as ck
    d, gs, T = 64, 64, 2
    f = Filled(lens, heads, d, gs, 32, torch.float16)
    at = offsets(lens)
    stretches = [(0, 1), (16, 32), (0, 1), (128, 700), (48, 64), (0, 1 << 30)]
    for b, n in enumerate(lens):
        a, e = (min(n, x) for x in stretches[b % len(stretches)])
        f.k[at[b] + a:at[b] + e, b % heads, 3] = (math.nan, math.inf, -math.inf)[b % 3]
    ck.kv4_append(f.cache, f.k, f.v, f.table, i32([0] * len(lens)), i32(at))
    q = rand_q(len(lens), T, 2 * heads, d, torch.float16)
    check_with_nan(ck.kv4_attention(q, f.cache, f.table, f.lengths), f.reference(q))


@pytest.mark.gpu
@pytest.mark.parametrize("n", [32, 33, 47, 700])
@pytest.mark.parametrize("T,group", [(1, 8), (1, 4), (2, 8)])
def test_nan_values_with_a_vanishing_weight_are_nan(n, T, group):
    """A weight below the smallest float is not 0 in the definition: NaN times it is NaN, in whole blocks and in those that need masks."""
    import crispybits_kernels as ck
    f = Filled([n, n], 1, 64, 32, 32, torch.float16)
    q = rand_q(2, T, group, 64, torch.float16).abs() + 0.5
    for b, t in ((0, 3), (1, n - 1 - T)):
        f.k[b * n + t] = -500.0                                    # scores some 3000 below the others
        f.v[b * n + t, 0, 40] = math.nan
    ck.kv4_append(f.cache, f.k, f.v, f.table, i32([0, 0]), i32([0, n, 2 * n]))
    got, (out, tol) = ck.kv4_attention(q, f.cache, f.table, f.lengths), f.reference(q)
    out[..., 32:] = math.nan
    check_with_nan(got, (out, tol))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,gain", [(torch.float16, 300.0), (torch.float16, 10000.0), (torch.bfloat16, 1e6), (torch.bfloat16, 1e12)])
@pytest.mark.parametrize("lens,heads", [([700, 33, 2500], 2), ([600, 5, 129] * 14, 4), ([100, 16, 33] * 50, 1)])
def test_scores_of_any_size(dtype, gain, lens, heads):
    """Queries and keys up to fp16's largest values and beyond: a row is the value of its best key, or the mean of those that share the best score.
    Scores are made of few bits, so that their fp32 sums are exact and neighbours 2^-6 of the largest apart, or equal."""
    import crispybits_kernels as ck
    d, n = 64, sum(lens)
    f = Filled(lens, heads, d, 64, 32, dtype)
    gen = torch.Generator().manual_seed(5)
    f.k.zero_()
    f.k[:, :, 0] = (torch.randint(1, 5, (n, heads), generator=gen) * 15 * 2.0 ** int(math.log2(gain) - 4)).to(dtype).to(DEV)   # code 15, a scale of few bits
    ck.kv4_append(f.cache, f.k, f.v, f.table, i32([0] * len(lens)), i32(offsets(lens)))
    q = torch.zeros(len(lens), 1, 2 * heads, d, dtype=dtype, device=DEV)
    q[..., 0] = 2.0 ** int(math.log2(gain))
    q[:, :, 1::2] *= -1
    got = ck.kv4_attention(q, f.cache, f.table, f.lengths)
    at, (vc, vs, vl) = offsets(lens), quantise64(f.v, 64)
    for b in range(len(lens)):
        for h in range(2 * heads):
            s = f.k[at[b]:at[b + 1], h // 2, 0].double() * q[b, 0, h, 0].double()
            best = (s == s.max()).nonzero()[:, 0] + at[b]
            val, step = values64(vc[best], vs[best], vl[best])[:, h // 2], vs[best][:, h // 2].repeat_interleave(64, -1)
            want = val.mean(0)
            # weights alike: 2^-11 of |code - 7.5| steps each for their rounding, 2^-20 of all magnitudes for the fp32 sums
            tol = torch.finfo(dtype).eps / 2 * 1.01 * want.abs() + (2.0 ** -11 * 1.01 + 2.0 ** -18) * 7.5 * step.mean(0) + 2.0 ** -18 * val.abs().mean(0) + 1e-7
            assert ((got[b, 0, h].double() - want).abs() <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [0.0, 1e-9, None])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_queries_of_zeros_and_a_scale_of_zero_weigh_all_keys_alike(scale, dtype):
    import crispybits_kernels as ck
    lens = [20, 333, 1, 64]
    f = Filled(lens, 2, 64, 32, 32, dtype)
    q = rand_q(4, 3, 8, 64, dtype)
    q[:, :, ::2] = 0.0
    q[:, 1] *= 2.0 ** -20
    check(ck.kv4_attention(q, f.cache, f.table, f.lengths, scale=scale), f.reference(q, scale))


@pytest.mark.gpu
@pytest.mark.parametrize("power", [110, 119, 120, 121, 127])
def test_the_largest_bfloat16_queries(power):
    """One value of q and k alone, so that scores are 2^(power - 63 - t) / 8 for token t: the first has all the weight, exactly."""
    import crispybits_kernels as ck
    n = 20
    f = Filled([n], 1, 64, 32, 32, torch.bfloat16)
    f.k.zero_()
    f.k[:, 0, 0] = 2.0 ** (-60 - torch.arange(n, device=DEV))
    ck.kv4_append(f.cache, f.k, f.v, f.table, i32([0]), i32([0, n]))
    q = torch.zeros(1, 1, 2, 64, dtype=torch.bfloat16, device=DEV)
    q[..., 0] = 2.0 ** power
    q[:, :, 1] *= -1                                               # the last token's is the largest score, and 2^(power - 83) / 8 above the next
    got = ck.kv4_attention(q, f.cache, f.table, f.lengths)
    codes, scale, lo = quantise64(f.v, 32)
    for h, t in ((0, 0), (1, n - 1)):
        want = values64(codes, scale, lo)[t, 0]
        tol = torch.finfo(torch.bfloat16).eps / 2 * 1.01 * want.abs() + 2.0 ** -20 * (15 * scale + lo.abs())[t, 0].repeat_interleave(32)
        assert ((got[0, 0, h].double() - want).abs() <= tol).all()


def test_a_scale_that_is_not_finite_is_refused():
    from crispybits_kernels import _C
    lib, c = _C._lib, _C._KV4Cache(256, 4, 2, 128, 64, 64, 1)
    s3, s6 = (ctypes.c_int64 * 3)(8, 8, 8), (ctypes.c_int64 * 6)(*[128] * 6)
    for scale in (math.nan, math.inf, -math.inf, 1e39):
        assert lib.cb_kv4_attention(ctypes.byref(c), 256, s3, 256, 2, 1, 4, 256, 2, 256, scale, 256, 1 << 20, 256, 1 << 30, 0) == 1
        assert b"scale" in lib.cb_last_error()
        assert lib.cb_prompt_attention(256, 256, 256, s6, 256, 4, 4, 2, 2, 64, 1, 256, 256, 1, scale, 1, 256, 1 << 20, 256, 1 << 40, 0) == 1
        assert b"scale" in lib.cb_last_error()


@pytest.mark.gpu
def test_a_scale_that_is_not_finite_is_refused_in_python():
    import crispybits_kernels as ck
    f = Filled([20], 2, 64, 32, 16, torch.float16)
    q = rand_q(1, 1, 4, 64, torch.float16)
    for scale in (math.nan, math.inf, 1e39):
        with pytest.raises(RuntimeError, match="scale"):
            ck.kv4_attention(q, f.cache, f.table, f.lengths, scale=scale)
        with pytest.raises(RuntimeError, match="scale"):
            ck.prompt_attention(q[0], q[0], q[0], i32([0, 1]), scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("group", [1, 2, 3, 5, 7, 8, 9, 13, 17])
@pytest.mark.parametrize("T", [1, 2, 3])
def test_tiles_with_rows_to_spare(group, T):
    """Fewer rows than a tile has, in whole blocks, blocks that the newest tokens see in part, and blocks that end inside."""
    import crispybits_kernels as ck
    lens = [2, 31, 32, 33, 800, 1311]
    f = Filled(lens, 2, 64, 32, 32, torch.float16, seed=group)
    q = rand_q(len(lens), T, 2 * group, 64, torch.float16)
    check(ck.kv4_attention(q, f.cache, f.table, f.lengths), f.reference(q))


def exact_codes(row, gs, dtype):
    """Codes, scale and lo of one row, in rational arithmetic."""
    from fractions import Fraction as Fr
    codes, scales, los = [], [], []
    for g in range(0, len(row), gs):
        x = [Fr(v) for v in row[g:g + gs]]
        lo, want = min(x), (max(x) - min(x)) / 15
        near = torch.tensor(float(want), dtype=torch.double).to(dtype)
        around = torch.stack((near, torch.nextafter(near, torch.tensor(0.0).to(dtype)), torch.nextafter(near, torch.tensor(math.inf).to(dtype)))).double().tolist()
        even = lambda v: torch.tensor(v, dtype=torch.double).to(dtype).view(torch.int16).item() & 1
        scale = min((Fr(v) for v in around if math.isfinite(v)), key=lambda v: (abs(v - want), even(float(v))))
        codes += [0 if scale == 0 else min(15, round((v - lo) / scale)) for v in x]                     # Fraction rounds half to even
        scales.append(float(scale)); los.append(float(lo))
    return codes, scales, los


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_codes_at_half_steps_beside_a_tiny_minimum(dtype):
    """A minimum some 2^-30 of the other values: what a float loses of x - lo, and of the range, decides the ties.  Every byte as defined."""
    import crispybits_kernels as ck
    d, gs = 64, 32
    tiny = (2.0 ** -24, 2.0 ** -22) if dtype == torch.float16 else (2.0 ** -30, 2.0 ** -100)
    ends = [(lo, top) for top in (15.0, 15.0 * 2 ** -6) for lo in (*tiny, *(-t for t in tiny))]
    if dtype == torch.float16:
        # ranges hi - lo beside 15 t, t half way between two scales: hi = 15 t - r, lo = -r (1 +- 2^-10) with r of one bit, 2^-15 or 2^-14 of hi
        # (bfloat16 has none that a float does not hold: 15 t has 13 bits, hi 8, so that r is 2^-12 of it or more and lo a multiple of 2^-19)
        fits = lambda v: torch.tensor(v, dtype=torch.double).to(dtype).double().item() == v
        found = [(-r * e, 15 * t - r) for k in range(1 << 10, 1 << 11) for t in [(2 * k + 1) * 2.0 ** -11] for r in (2.0 ** -12, 2.0 ** -11, 2.0 ** -10)
                 if fits(15 * t - r) for e in (1 + 2.0 ** -10, 1 - 2.0 ** -11, 1.0)]
        assert len(found) >= 30
        ends += found[:12] + found[-12:]
    rows = []
    for lo, top in ends:
        step = torch.tensor((top - lo) / 15, dtype=torch.double).to(dtype).double().item()
        x = [lo, top, *((i + 0.5) * step for i in range(15))]
        rows.append((x + [1.0 * step] * (gs - len(x))) * 2)
    x = torch.tensor(rows, dtype=torch.double).to(dtype)
    x[:, gs:] *= -1
    n = x.shape[0]
    c = ck.KV4Cache.empty(1, 1, d, 64, gs, dtype)
    c.pages.zero_()
    xs = x[:, None].to(DEV)
    ck.kv4_append(c, xs, xs, i32([[0]]), i32([0]), i32([0, n]))
    page, lay = torch.zeros(c.pages.shape[2], dtype=torch.uint8), Layout(d, gs)
    for i in range(n):
        codes, scale, lo = exact_codes(x[i].double().tolist(), gs, dtype)
        for which in "kv":
            lay.put(page, which, i, codes, torch.tensor(scale), torch.tensor(lo), dtype)
    got = c.pages[0, 0].cpu()
    assert torch.equal(got, page), f"{int((got != page).sum())} bytes differ"


@pytest.mark.gpu
@pytest.mark.parametrize("gs", [32, 64])
def test_groups_whose_range_is_no_float(gs):
    """Finite bfloat16 values more than the largest float apart: bytes as defined, and values read back (those beyond the largest are the largest)."""
    import crispybits_kernels as ck
    d, top = 64, torch.finfo(torch.bfloat16).max
    gen = torch.Generator().manual_seed(1)
    rows = [torch.linspace(-1, 1, d, dtype=torch.double) * top, torch.where(torch.rand(d, generator=gen) < 0.5, -top, top).double(),
            torch.cat((torch.full((63,), -top), torch.tensor([2.0 ** -133]))).double(), (torch.rand(d, generator=gen).double() * 2 - 1) * top,
            (torch.rand(d, generator=gen).double() * 1.1 - 0.1) * top, torch.tensor([-top, top, *(-top + (i % 15 + 0.5) * (top / 7.5) for i in range(62))]),
            torch.tensor([-top * 0.51, top * 0.51, *([1.0, -2.0 ** -133] * 31)])]
    x = torch.stack([r.double() for r in rows]).to(torch.bfloat16)
    x = torch.where(torch.isfinite(x), x, torch.tensor(top).to(x.dtype))
    x = torch.cat((x, -x))
    n = x.shape[0]
    c = ck.KV4Cache.empty(1, 1, d, 64, gs, torch.bfloat16)
    c.pages.zero_()
    xs = x[:, None].to(DEV)
    ck.kv4_append(c, xs, xs, i32([[0]]), i32([0]), i32([0, n]))
    page, lay, want = torch.zeros(c.pages.shape[2], dtype=torch.uint8), Layout(d, gs), []
    for i in range(n):
        codes, scale, lo = exact_codes(x[i].double().tolist(), gs, torch.bfloat16)
        want.append([k * scale[j // gs] + lo[j // gs] for j, k in enumerate(codes)])
        for which in "kv":
            lay.put(page, which, i, codes, torch.tensor(scale, dtype=torch.double), torch.tensor(lo, dtype=torch.double), torch.bfloat16)
    got = c.pages[0, 0].cpu()
    assert torch.equal(got, page), f"{int((got != page).sum())} bytes differ"
    want = torch.tensor(want, dtype=torch.double).clamp(-top, top)
    for y in ck.kv4_read(c, i32([[0]]), i32([0]), i32([0, n]), n):
        # one rounding of the type, of a sum of two that fp32 may have rounded first
        assert ((y[:, 0].cpu().double() - want).abs() <= want.abs() * (2.0 ** -8 + 2.0 ** -20) + 2.0 ** -24 * 2 * top + 2.0 ** -133).all()


@pytest.mark.gpu
def test_counters_left_by_a_launch_that_gave_up_are_zeroed_with_its_status(monkeypatch):
    """A launch that gives up leaves counts behind.  They are planted here, with the status that such a launch sets: once the status is read, eager and
    captured calls are right again."""
    import crispybits_kernels as ck
    from crispybits_kernels import _C
    f = Filled([3000, 40, 900], 2, 64, 64, 64, torch.float16)
    q, cu = rand_q(3, 1, 4, 64, torch.float16), i32([0, 300])
    pq, pk, cu_k = rand_kv(300, 4, 64, torch.float16, 1), rand_kv(9300, 2, 64, torch.float16, 2), i32([0, 9300])

    def both():
        return ck.kv4_attention(q, f.cache, f.table, f.lengths), ck.prompt_attention(pq, pk, pk, cu, cu_k)

    want = both()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = both()
    torch.cuda.synchronize()
    dev = torch.cuda.current_device()
    for (d, _), have in _C._attention_eager.items():
        if d == dev:
            have[0].fill_(1)
    _C._attention_slab[dev][0].fill_(1)
    with monkeypatch.context() as m:
        def status(out):
            out._obj.value = 3002
            return 0
        m.setattr(_C._lib, "cb_decode_status", status)
        assert _C.decode_status() == 3002
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(both(), want))
        g.replay()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
    assert _C.decode_status() == 0


@pytest.mark.gpu
def test_calls_of_different_needs_share_scratch_without_making_it_anew():
    """Many counters and little scratch, then the other way round: after one round of both nothing is allocated any more."""
    import crispybits_kernels as ck
    from crispybits_kernels import _C
    B, heads = 260, 40                                             # 10400 counters
    f = Filled([1] * B, heads, 64, 64, 16, torch.float16)
    q, x, cu = rand_q(B, 1, heads, 64, torch.float16), rand_kv(2000, 2, 128, torch.float16, 1), i32([0, 2000])
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        kept = []
        for _ in range(3):
            ck.kv4_attention(q, f.cache, f.table, f.lengths)
            ck.prompt_attention(x, x, x, cu)
            have = _C._attention_eager[(torch.cuda.current_device(), s.cuda_stream)]
            kept.append([t.data_ptr() for t in have])
            assert have[0].numel() >= B * heads
    torch.cuda.synchronize()
    assert kept[0] == kept[1] == kept[2]


# ------------------------------------------------------------------------------------------------ GPU: each schedule against the definition
def schedule(lens, heads, rows):
    """How kv4_attention shares out the work: ("aligned" parts that end with their segments, or "equal" ones that cut them), and whether short segments
    go to single warps."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    segs = heads * (-(-rows // (16 if rows > 8 else 8)))
    blocks, total = segs * sum(-(-n // 16) for n in lens), len(lens) * segs
    if 4 * total <= sms and not (16 * total > sms and blocks > 16 * sms):
        return "aligned", False
    return "equal", 4 * total > sms and total >= sms


def mixed(count, pattern):
    return [pattern[i % len(pattern)] for i in range(count)]


SCHEDULES = [(mixed(5, [1000, 0, 3, 700, 64]), 2, 1, 1, ("aligned", False)), (mixed(20, [900, 1, 333, 0, 64, 1000, 17, 500]), 4, 1, 4, ("equal", False)),
             (mixed(25, [129, 700, 0, 1, 40]), 4, 2, 2, ("equal", False)), (mixed(40, [100, 1, 129, 0, 2000, 128]), 4, 1, 1, ("equal", True)),
             (mixed(70, [5, 2000, 130, 100]), 3, 3, 4, ("equal", True)), ([1500, 1600, 1700, 1540, 1499, 2100, 1800, 1650], 4, 1, 2, ("equal", False)),
             ([4000, 3900], 6, 2, 3, ("equal", False)), ([3000] * 37, 1, 1, 9, ("equal", False))]


@pytest.mark.gpu
@pytest.mark.parametrize("lens,heads,T,group,kind", SCHEDULES)
@pytest.mark.parametrize("d,gs,dtype", [(64, 32, torch.bfloat16), (128, 64, torch.float16)])
def test_each_schedule_matches_the_definition(lens, heads, T, group, kind, d, gs, dtype):
    """Parts joined across cuts, single warps and cut segments in one launch, the device's own change from aligned to equal parts."""
    import crispybits_kernels as ck
    if torch.cuda.get_device_properties(0).multi_processor_count == 148:
        assert schedule(lens, heads, T * group) == kind
    f = Filled(lens, heads, d, gs, 16, dtype, seed=len(lens))
    q = rand_q(len(lens), T, heads * group, d, dtype)
    got = ck.kv4_attention(q, f.cache, f.table, f.lengths)
    check(got, f.reference(q))
    assert torch.equal(got, ck.kv4_attention(q, f.cache, f.table, f.lengths))
