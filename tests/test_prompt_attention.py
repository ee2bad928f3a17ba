"""Attention of packed prompts against softmax(scale * q K^T) V in 64 bits."""
import ctypes
import math

import pytest
import torch

DEV = "cuda"


# ------------------------------------------------------------------------------------------------ refusals, no GPU needed
def test_c_entry_point_refuses_bad_arguments():
    from crispybits_kernels import _C
    lib, s6 = _C._lib, (ctypes.c_int64 * 6)(*[128] * 6)

    def call(q=256, k=256, v=256, st=s6, out=256, tq=4, tk=4, h=2, hkv=2, d=64, dt=1, cq=256, ck=256, b=1, cnt=256, part=256):
        return lib.cb_prompt_attention(q, k, v, st, out, tq, tk, h, hkv, d, dt, cq, ck, b, 1.0, 1, cnt, 1 << 20, part, 1 << 40, 0)

    for bad in (dict(dt=0), dict(dt=3), dict(d=96), dict(d=256), dict(tq=-1), dict(tk=-1), dict(tq=1 << 30), dict(h=3), dict(hkv=0), dict(b=-1),
                dict(q=0), dict(k=0), dict(v=0), dict(out=0), dict(cq=0), dict(ck=0), dict(st=None), dict(q=8), dict(k=8), dict(v=8),
                dict(out=8), dict(cnt=0), dict(part=0), dict(part=8), dict(st=(ctypes.c_int64 * 6)(128, 128, 128, 4, 128, 128)), dict(st=(ctypes.c_int64 * 6)(0, *[128] * 5)),
                dict(st=(ctypes.c_int64 * 6)(128, 128, -128, 128, 128, 128))):
        assert call(**bad) == 1 and lib.cb_last_error(), bad
    assert call(tq=0) == 0 and call(b=0) == 0 and call(h=0) == 0


def test_c_entry_point_refuses_an_output_on_its_inputs():
    """Other rows may still be read while one is written."""
    from crispybits_kernels import _C
    lib, s6 = _C._lib, (ctypes.c_int64 * 6)(256, 64, 128, 64, 128, 64)
    size = 4 * 256 * 2                                          # 4 queries of 4 heads (k and v: 4 keys of 2 heads), 64 values
    q, k, v, out, far = 1 << 20, 2 << 20, 3 << 20, 4 << 20, 1 << 30

    def message(out):
        assert lib.cb_prompt_attention(q, k, v, s6, out, 4, 4, 4, 2, 64, 1, far, far, 1, 1.0, 1, far, 1 << 30, far, 1 << 40, 0) != 0
        return lib.cb_last_error().decode()

    for near in (q, q + size - 16, q - size + 16, k, k + 1024 - 16, v - size + 16):
        assert "shares memory" in message(near), near
    if not torch.cuda.is_available():                           # (nothing is launched without a device)
        for apart in (out, q + size, q - size, k + 1024, v - size):
            assert "shares memory" not in message(apart), apart


def test_python_entry_point_refuses_cpu_tensors():
    import crispybits_kernels as ck
    x = torch.zeros(2, 2, 64).half()
    with pytest.raises(RuntimeError):
        ck.prompt_attention(x, x, x, torch.tensor([0, 2], dtype=torch.int32))


# ------------------------------------------------------------------------------------------------ GPU
def i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def offsets(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def rand(n, heads, d, dtype, seed, gain=1.0):
    return (torch.randn(n, heads, d, generator=torch.Generator().manual_seed(seed)) * gain).to(dtype).to(DEV)


def reference(q, k, v, cu_q, cu_k, scale=None, causal=True):
    """(out, tolerance) in 64 bits.

    Tolerance: the output's rounding, eps / 2 of it; the weights' rounding to the inputs' type, eps / 2 of each, so eps / 2 of
    sum w |v|; the scores' fp32 sums (2^-20 of sum |q| |k| is ample for 128 products) and the exponential (2^-21), which move
    each weight and their sum."""
    D, share = q.shape[2], q.shape[1] // k.shape[1]
    scale = D ** -0.5 if scale is None else scale
    out, tol = torch.zeros(q.shape, dtype=torch.double, device=DEV), torch.zeros(q.shape, dtype=torch.double, device=DEV)
    half = torch.finfo(q.dtype).eps / 2
    for b in range(len(cu_q) - 1):
        (q0, q1), (k0, k1) = cu_q[b:b + 2], cu_k[b:b + 2]
        if q1 <= q0 or k1 <= k0:
            continue
        qq = q[q0:q1].double().transpose(0, 1)
        kk, vv = (x[k0:k1].double().transpose(0, 1).repeat_interleave(share, 0) for x in (k, v))
        s = qq @ kk.transpose(1, 2) * scale
        err = 2.0 ** -20 * (qq.abs() @ kk.abs().transpose(1, 2)) * abs(scale)
        if causal:
            hidden = torch.arange(k1 - k0, device=DEV)[None] > torch.arange(q1 - q0, device=DEV)[:, None] + (k1 - k0) - (q1 - q0)
            s, err = s.masked_fill(hidden, -math.inf), err.masked_fill(hidden, 0)
        w = torch.softmax(s, -1).nan_to_num(0.0)
        o, size = w @ vv, w @ vv.abs()
        e = err.amax(-1, keepdim=True) + 2.0 ** -21
        out[q0:q1] = o.transpose(0, 1)
        tol[q0:q1] = (half * o.abs() * 1.01 + (half * 1.01 + 2 * e) * size + 1e-7).transpose(0, 1)
    return out, tol


def check(got, want):
    out, tol = want
    over = (got.double() - out).abs() - tol
    assert torch.isfinite(got).all() and (over <= 0).all(), f"{over.max():.2e} over, at tolerance {tol[over == over.max()][0]:.2e}"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n", [1, 2, 63, 64, 127, 128, 129, 255, 256, 257, 300, 1000])
def test_one_prompt(dtype, d, n):
    import crispybits_kernels as ck
    q, k, v = rand(n, 4, d, dtype, 1), rand(n, 2, d, dtype, 2), rand(n, 2, d, dtype, 3)
    check(ck.prompt_attention(q, k, v, i32([0, n])), reference(q, k, v, [0, n], [0, n]))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d,heads,kv", [(128, 6, 2), (64, 5, 5), (64, 8, 1)])
@pytest.mark.parametrize("causal", [True, False])
def test_packed_prompts_with_and_without_a_past(dtype, d, heads, kv, causal):
    """Lengths from none to several tiles; keys more, as many, and fewer than queries (rows that see none), and none at all."""
    import crispybits_kernels as ck
    lens = [5, 0, 1, 300, 128, 513, 40, 7, 130]
    keys = [5, 9, 700, 300, 385, 520, 33, 0, 2]
    cq, ckv = offsets(lens), offsets(keys)
    q, k, v = rand(cq[-1], heads, d, dtype, 1), rand(ckv[-1], kv, d, dtype, 2), rand(ckv[-1], kv, d, dtype, 3)
    got = ck.prompt_attention(q, k, v, i32(cq), i32(ckv), causal=causal)
    check(got, reference(q, k, v, cq, ckv, causal=causal))
    assert (got[cq[7]:cq[8]] == 0).all()                       # no keys
    if causal:
        assert (got[cq[6]:cq[6] + 7] == 0).all() and (got[cq[8]:cq[8] + 128] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("B", [31, 32, 33, 200])
def test_many_prompts(B):
    """More sequences than a warp looks at together, more tiles than SMs."""
    import crispybits_kernels as ck
    lens = [(37 * b) % 90 + (500 if b % 17 == 3 else 0) for b in range(B)]
    cu = offsets(lens)
    q, k, v = rand(cu[-1], 2, 64, torch.float16, 1), rand(cu[-1], 1, 64, torch.float16, 2), rand(cu[-1], 1, 64, torch.float16, 3)
    check(ck.prompt_attention(q, k, v, i32(cu)), reference(q, k, v, cu, cu))


@pytest.mark.gpu
def test_a_long_prompt_and_rising_scores():
    """Keys that grow along the sequence, so that the running maximum moves at almost every tile."""
    import crispybits_kernels as ck
    n = 3000
    for dtype in (torch.float16, torch.bfloat16):
        q, k, v = rand(n, 2, 128, dtype, 1, 2.0), rand(n, 2, 128, dtype, 2), rand(n, 2, 128, dtype, 3)
        k = (k.float() * torch.linspace(0.02, 3.0, n, device=DEV)[:, None, None]).to(dtype)
        check(ck.prompt_attention(q, k, v, i32([0, n])), reference(q, k, v, [0, n], [0, n]))
        k = k.flip(0).contiguous()
        check(ck.prompt_attention(q, k, v, i32([0, n])), reference(q, k, v, [0, n], [0, n]))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,d,causal", [(torch.float16, 64, True), (torch.bfloat16, 128, True), (torch.float16, 128, False)])
@pytest.mark.parametrize("lens,past", [([300], [9000]), ([1], [4096]), ([130, 0, 257, 5], [5000, 700, 0, 6001]), ([3000], [0]), ([64, 64], [3968, 0])])
def test_keys_cut_into_parts(dtype, d, causal, lens, past):
    """Few tiles over many keys: their keys are shared out among the SMs."""
    import crispybits_kernels as ck
    cq, ckv = offsets(lens), offsets([n + p for n, p in zip(lens, past)])
    q, k, v = rand(cq[-1], 4, d, dtype, 1), rand(ckv[-1], 2, d, dtype, 2), rand(ckv[-1], 2, d, dtype, 3)
    k = (k.float() * torch.linspace(0.1, 2.0, ckv[-1], device=DEV)[:, None, None]).to(dtype)
    want = reference(q, k, v, cq, ckv, causal=causal)
    first = ck.prompt_attention(q, k, v, i32(cq), i32(ckv), causal=causal)
    check(first, want)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for s in streams * 3:
        with torch.cuda.stream(s):
            outs.append(ck.prompt_attention(q, k, v, i32(cq), i32(ckv), causal=causal))
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        a, b = i32(cq), i32(ckv)
        with torch.cuda.graph(g):
            outs.append(ck.prompt_attention(q, k, v, a, b, causal=causal))
        graphs.append((g, a, b))
    for _ in range(3):
        for (g, *_), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(first, o) for o in outs)


@pytest.mark.gpu
def test_bounds_that_overlap():
    """Sequences that name the same rows again and again: more tiles than the rows make."""
    import crispybits_kernels as ck
    n = 3000
    q, k, v = rand(n, 1, 64, torch.float16, 1), rand(4 * n, 1, 64, torch.float16, 2), rand(4 * n, 1, 64, torch.float16, 3)
    B = 11
    cu, cu_k = i32([0, n] * (B // 2) + [0, n]), i32([0, 4 * n] * (B // 2) + [0, 4 * n])
    got = ck.prompt_attention(q, k, v, cu, cu_k, causal=False)
    check(got, reference(q, k, v, [0, n], [0, 4 * n], causal=False))


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [0.25, -0.1, 0.0])
def test_scale(scale):
    import crispybits_kernels as ck
    q, k, v = rand(200, 2, 64, torch.bfloat16, 1), rand(200, 2, 64, torch.bfloat16, 2), rand(200, 2, 64, torch.bfloat16, 3)
    check(ck.prompt_attention(q, k, v, i32([0, 200]), scale=scale), reference(q, k, v, [0, 200], [0, 200], scale))


@pytest.mark.gpu
def test_strides_and_alignment():
    import crispybits_kernels as ck
    n, d = 150, 64
    fused = rand(n, 8, d, torch.float16, 1).flatten(1)          # [q: 4 heads | k: 2 | v: 2]
    q, k, v = fused[:, :4 * d].view(n, 4, d), fused[:, 4 * d:6 * d].view(n, 2, d), fused[:, 6 * d:].view(n, 2, d)
    cu = i32([0, n])
    want = ck.prompt_attention(q.contiguous(), k.contiguous(), v.contiguous(), cu)
    check(want, reference(q, k, v, [0, n], [0, n]))
    assert torch.equal(want, ck.prompt_attention(q, k, v, cu))
    heads_first = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v)]
    assert torch.equal(want, ck.prompt_attention(*heads_first, cu))
    odd = torch.empty(q.numel() + 1, dtype=q.dtype, device=DEV)[1:].view(q.shape).copy_(q)
    assert torch.equal(want, ck.prompt_attention(odd, k, v, cu))
    one = k[:, :1].expand(n, 2, d)                              # a head shared by expanding it
    assert torch.equal(ck.prompt_attention(q, one, one, cu), ck.prompt_attention(q, k[:, :1], k[:, :1], cu))
    assert torch.equal(ck.prompt_attention(q[:1], k[:1], v[:1], i32([0, 1])), v[:1].repeat_interleave(2, 1))


@pytest.mark.gpu
def test_rows_of_no_sequence_and_values_of_others():
    """Rows before the first and behind the last sequence stay; infinities and NaN of other rows do not reach a sequence."""
    import crispybits_kernels as ck
    n, d = 700, 128
    q, k, v = rand(n, 2, d, torch.bfloat16, 1), rand(n, 1, d, torch.bfloat16, 2), rand(n, 1, d, torch.bfloat16, 3)
    cu = [100, 233, 233, 600]
    want = reference(q, k, v, cu, cu)
    for x in (q, k, v):
        x[:100] = math.nan
        x[600:650] = math.inf
        x[650:] = math.nan
    out = torch.full((n, 2, d), 7.0, dtype=torch.bfloat16, device=DEV)
    got = ck.prompt_attention(q, k, v, i32(cu), out=out)
    assert got is out and (out[:100] == 7).all() and (out[600:] == 7).all()
    check(out[100:600], tuple(t[100:600] for t in want))
    # keys of their own bounds, with NaN directly behind them
    k[333:], v[333:] = math.nan, math.nan
    got = ck.prompt_attention(q[100:300], k, v, i32([0, 200]), i32([150, 333]), causal=False)
    check(got, reference(q[100:300], k, v, [0, 200], [150, 333], causal=False))
    # bounds outside the tensors are cut to them
    got = ck.prompt_attention(q[100:300], k[:333], v[:333], i32([-5, 10000]), i32([100, 1 << 30]), causal=False)
    check(got, reference(q[100:300], k, v, [0, 200], [100, 333], causal=False))


@pytest.mark.gpu
def test_nan_in_a_sequence_reaches_only_that_sequence():
    import crispybits_kernels as ck
    cu = [0, 70, 140, 210]
    q, k, v = (rand(210, 1, 64, torch.float16, s) for s in (1, 2, 3))
    want = ck.prompt_attention(q, k, v, i32(cu))
    k[100] = math.nan
    got = ck.prompt_attention(q, k, v, i32(cu))
    assert torch.equal(got[:100], want[:100]) and torch.equal(got[140:], want[140:]) and got[100:140].isnan().all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n,past", [(300, 0), (200, 65), (130, 3000), (700, -40)])
def test_values_that_are_not_finite_reach_the_queries_that_see_them(dtype, d, n, past):
    """An infinity or a NaN in v, anywhere: queries before it are what they are without it, later ones are not finite in that value only."""
    import crispybits_kernels as ck
    cq, ckv = [0, n, n + 50], [0, n + past, n + past + 50]
    q, k, v = rand(cq[-1], 2, d, dtype, 1), rand(ckv[-1], 1, d, dtype, 2), rand(ckv[-1], 1, d, dtype, 3)
    gen = torch.Generator().manual_seed(n)
    spots = [(int(torch.randint(0, n + past, (1,), generator=gen)), int(torch.randint(0, d, (1,), generator=gen))) for _ in range(5)]
    spots += [(n + past - 1, 0), (max(0, n + past - 129), d - 1)]
    bad = v.clone()
    for i, (key, col) in enumerate(spots):
        v[key, 0, col] = 0
        bad[key, 0, col] = (math.nan, math.inf, -math.inf)[i % 3]
    want, tol = reference(q, k, v, cq, ckv)
    got = ck.prompt_attention(q, k, bad, i32(cq), i32(ckv))
    hit = torch.zeros(cq[-1], 2, d, dtype=torch.bool, device=DEV)
    for key, col in spots:
        hit[max(0, key - past):n, :, col] = True
    assert torch.equal(~torch.isfinite(got), hit)
    assert ((got.double() - want).abs() <= tol)[~hit].all()      # a sum formed again has fewer roundings, not more


@pytest.mark.gpu
def test_the_same_every_time_on_any_stream_and_captured():
    import crispybits_kernels as ck
    from crispybits_kernels import _C
    cu = offsets([900, 30, 1400, 128])
    q, k, v = rand(cu[-1], 8, 128, torch.bfloat16, 1), rand(cu[-1], 2, 128, torch.bfloat16, 2), rand(cu[-1], 2, 128, torch.bfloat16, 3)
    c = i32(cu)
    want = ck.prompt_attention(q, k, v, c)
    check(want, reference(q, k, v, cu, cu))
    torch.cuda.synchronize()
    outs = []
    for s in [torch.cuda.Stream() for _ in range(3)] * 3:
        with torch.cuda.stream(s):
            outs.append(ck.prompt_attention(q, k, v, c))
    torch.cuda.synchronize()
    assert all(torch.equal(want, o) for o in outs)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ck.prompt_attention(q, k, v, c)
    for cu2 in ([0, 1, 2, 3, cu[-1]], cu):                       # a replay reads what the bounds hold then
        c.copy_(i32(cu2))
        g.replay()
        check(out, reference(q, k, v, cu2, cu2))
    assert torch.equal(out, want) and _C.decode_status() == 0


@pytest.mark.gpu
def test_refusals_on_the_device():
    import crispybits_kernels as ck
    q, k = rand(10, 4, 64, torch.float16, 1), rand(10, 2, 64, torch.float16, 2)
    cu = i32([0, 10])
    for args in ((q.float(), k.float(), k.float(), cu), (q, k.bfloat16(), k, cu), (q, k, k[:, :1], cu), (q[:, :3], k, k, cu), (q, k.cpu(), k, cu),
                 (q[..., :32], k[..., :32], k[..., :32], cu), (q[0], k, k, cu), (q, k, k, cu.long()), (q, k, k, cu.cpu()), (q, k, k, cu[None]),
                 (q, k, k, cu, i32([0, 5, 10]))):
        with pytest.raises(RuntimeError):
            ck.prompt_attention(*args)
    for out in (torch.empty(10, 4, 64, device=DEV), torch.empty(10, 4, 128, device=DEV, dtype=q.dtype)[..., :64], torch.empty(9, 4, 64, device=DEV, dtype=q.dtype)):
        with pytest.raises(RuntimeError):
            ck.prompt_attention(q, k, k, cu, out=out)
    both = torch.zeros(2, 10, 4, 64, device=DEV, dtype=q.dtype)
    for out in (q, both.view(20, 4, 64)[5:15]):
        with pytest.raises(RuntimeError, match="shares memory"):
            ck.prompt_attention(q if out is q else both[0], k, k, cu, out=out)
    assert (ck.prompt_attention(both[0], k, k, cu, out=both[1]) == ck.prompt_attention(both[0], k, k, cu)).all()
    assert ck.prompt_attention(q[:0], k, k, i32([0, 0])).shape == (0, 4, 64)
    none = ck.prompt_attention(q, k[:0], k[:0], cu, i32([0, 0]))
    assert (none == 0).all()


# ------------------------------------------------------------------------------------------------ GPU: queries and keys that are not finite
def check_with_nan(got, want):
    """NaN exactly where the definition has NaN, everything else within its tolerance."""
    out, tol = want
    assert torch.equal(got.isnan(), out.isnan()), f"{int((got.isnan() != out.isnan()).sum())} of {got.numel()} values"
    there = ~out.isnan()
    assert ((got.double() - out).abs() <= tol)[there].all() and torch.isfinite(got[there]).all()


def reference_with_nan(q, k, v, cu_q, cu_k, causal=True):
    """`reference`, with NaN where a row that sees a key has a score that is NaN, two that are +inf, or none above -inf.  Its tolerance is formed of the
    weights w that these scores give: sum w |v| is another where a key of score -inf has none.  The scores' error is that of the finite keys."""
    def finite(x):
        return torch.where(torch.isfinite(x), x, 0).double()
    share, half = q.shape[1] // k.shape[1], torch.finfo(q.dtype).eps / 2
    out, tol = torch.zeros(q.shape, dtype=torch.double, device=DEV), torch.zeros(q.shape, dtype=torch.double, device=DEV)
    for b in range(len(cu_q) - 1):
        (q0, q1), (k0, k1) = cu_q[b:b + 2], cu_k[b:b + 2]
        if q1 <= q0 or k1 <= k0:
            continue
        qq = q[q0:q1].transpose(0, 1)
        kk, vv = (x[k0:k1].transpose(0, 1).repeat_interleave(share, 0) for x in (k, v))
        s = qq.double() @ kk.double().transpose(1, 2) * q.shape[2] ** -0.5
        err = 2.0 ** -20 * (finite(qq).abs() @ finite(kk).abs().transpose(1, 2)) * q.shape[2] ** -0.5
        hidden = torch.zeros(s.shape[1:], dtype=torch.bool, device=DEV)
        if causal:
            hidden = torch.arange(k1 - k0, device=DEV)[None] > torch.arange(q1 - q0, device=DEV)[:, None] + (k1 - k0) - (q1 - q0)
        w = torch.softmax(s.masked_fill(hidden, -math.inf), -1)
        w = torch.where(hidden.all(-1)[None, :, None], 0.0, w)
        o, e = w @ vv.double(), err.masked_fill(hidden, 0).amax(-1, keepdim=True) + 2.0 ** -21
        out[q0:q1] = o.transpose(0, 1)
        tol[q0:q1] = (half * o.abs() * 1.01 + (half * 1.01 + 2 * e) * (w @ vv.double().abs()) + 1e-7).transpose(0, 1)
    return out, tol


# whole tiles, tiles cut into parts, and both; keys fewer than queries among them
NON_FINITE_SHAPES = [([300], [0]), ([130, 5], [6000, 700]), ([513, 70, 40, 1], [0, 3000, -10, 9000]), ([1], [0])]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,d", [(torch.float16, 64), (torch.bfloat16, 128)])
@pytest.mark.parametrize("lens,past", NON_FINITE_SHAPES)
@pytest.mark.parametrize("causal", [True, False])
def test_queries_that_are_not_finite_give_nan_wherever_the_work_is_cut(dtype, d, lens, past, causal):
    import crispybits_kernels as ck
    cq, ckv = offsets(lens), offsets([n + p for n, p in zip(lens, past)])
    q, k, v = rand(cq[-1], 4, d, dtype, 1), rand(ckv[-1], 2, d, dtype, 2), rand(ckv[-1], 2, d, dtype, 3)
    k[:, :, 9] = k[:, :, 9].abs() + 0.125                            # an infinity in q's value 9 makes all scores one infinity
    for i, r in enumerate(sorted({0, cq[-1] - 1, *cq[1:-1], *(c - 1 for c in cq[1:])} - {cq[-1]})):
        q[r, i % 4, 9] = (math.nan, math.inf, -math.inf)[i % 3]
        q[r, (i + 1) % 4, 20] = (-math.inf, math.nan, math.inf)[i % 3]
    want = reference_with_nan(q, k, v, cq, ckv, causal)
    assert want[0].isnan().any()
    check_with_nan(ck.prompt_attention(q, k, v, i32(cq), i32(ckv), causal=causal), want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,d", [(torch.float16, 128), (torch.bfloat16, 64)])
@pytest.mark.parametrize("lens,past", NON_FINITE_SHAPES)
@pytest.mark.parametrize("first,last", [(0, 1), (0, 128), (2, 1 << 30), (100, 1400), (0, 1 << 30)])
def test_keys_that_are_not_finite_wherever_the_work_is_cut(dtype, d, lens, past, first, last):
    """NaN keys make the rows that see them NaN; scores of -inf have no weight, and a row that has no others is NaN."""
    import crispybits_kernels as ck
    cq, ckv = offsets(lens), offsets([n + p for n, p in zip(lens, past)])
    q, k, v = rand(cq[-1], 2, d, dtype, 1), rand(ckv[-1], 2, d, dtype, 2), rand(ckv[-1], 2, d, dtype, 3)
    q[:, :, 5] = q[:, :, 5].abs() + 0.125
    for b, (a, e) in enumerate(zip(ckv, ckv[1:])):
        k[min(a + first, e):min(a + last, e), 0, 5] = math.nan
        k[min(a + first, e):min(a + last, e), 1, 5] = -math.inf      # scores of -inf for every query
    want = reference_with_nan(q, k, v, cq, ckv)
    check_with_nan(ck.prompt_attention(q, k, v, i32(cq), i32(ckv)), want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,gain", [(torch.float16, 300.0), (torch.float16, 10000.0), (torch.bfloat16, 1e6), (torch.bfloat16, 1e12)])
@pytest.mark.parametrize("n,past", [(300, 0), (130, 6000)])
@pytest.mark.parametrize("scale", [None, -0.125])
def test_scores_of_any_size(dtype, gain, n, past, scale):
    """Queries and keys up to fp16's largest values and beyond: a row is the value of its best key, or the mean of those that share the best score.
    Scores are made of few bits, so that they are exact, and neighbours are 1/4 of the largest apart, or equal."""
    import crispybits_kernels as ck
    gen = torch.Generator().manual_seed(5)
    q, k, v = torch.zeros(n, 2, 64, dtype=dtype, device=DEV), torch.zeros(n + past, 1, 64, dtype=dtype, device=DEV), rand(n + past, 1, 64, dtype, 3)
    power = 2.0 ** int(math.log2(gain))
    k[:, 0, 0] = (torch.randint(1, 5, (n + past,), generator=gen) * power).to(dtype).to(DEV)
    q[:, 0, 0], q[:, 1, 0] = power, -power
    got = ck.prompt_attention(q, k, v, i32([0, n]), i32([0, n + past]), scale=scale)
    s = torch.einsum("qh,k->hqk", q[:, :, 0].double(), k[:, 0, 0].double()) * (0.125 if scale is None else scale)
    s = s.masked_fill(torch.arange(n + past, device=DEV)[None] > torch.arange(n, device=DEV)[:, None] + past, -math.inf)
    w = (s == s.amax(-1, keepdim=True)).double()
    w /= w.sum(-1, keepdim=True)
    want, size = (torch.einsum("hqk,kd->qhd", w, x) for x in (v[:, 0].double(), v[:, 0].double().abs()))
    half = torch.finfo(dtype).eps / 2
    assert ((got.double() - want).abs() <= half * 1.01 * want.abs() + (half * 1.01 + 2.0 ** -18) * size + 1e-7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("n,past", [(200, 0), (100, 5000)])
def test_a_scale_of_zero_weighs_large_keys_alike_too(n, past):
    """Scores of up to 2^120, times a scale of 0: each row is the mean of the values that it sees."""
    import crispybits_kernels as ck
    cq, ckv = [0, n], [0, n + past]
    q, k, v = rand(n, 2, 64, torch.bfloat16, 1, 2.0 ** 56), rand(n + past, 1, 64, torch.bfloat16, 2, 2.0 ** 56), rand(n + past, 1, 64, torch.bfloat16, 3)
    got = ck.prompt_attention(q, k, v, i32(cq), i32(ckv), scale=0.0)
    check(got, reference(torch.zeros_like(q), k, v, cq, ckv, 0.0))


@pytest.mark.gpu
@pytest.mark.parametrize("d,dtype", [(64, torch.float16), (128, torch.bfloat16)])
def test_a_value_that_is_not_finite_behind_very_many_keys(d, dtype):
    """The rows before it form their sums again over tens of thousands of keys each; who waits for them meanwhile does not give up."""
    import crispybits_kernels as ck
    from crispybits_kernels import _C
    n = 131072
    q, k, v = rand(n, 1, d, dtype, 1), rand(n, 1, d, dtype, 2), rand(n, 1, d, dtype, 3)
    spots = [(n - 70, 3, math.nan), (n - 60, d - 1, math.inf), (60000, 17, -math.inf)]
    clean = v.clone()
    for key, col, x in spots:
        clean[key, 0, col], v[key, 0, col] = 0.0, x
    _C.decode_status()
    got = ck.prompt_attention(q, k, v, i32([0, n]))
    assert _C.decode_status() == 0
    hit = torch.zeros(n, 1, d, dtype=torch.bool, device=DEV)
    for key, col, _ in spots:
        hit[key:, :, col] = True
    assert torch.equal(~torch.isfinite(got), hit)
    for a in (n - 256, n - 128, 59904):                              # sequences that end with the rows of a tile: the same rows, from their definition
        want, tol = reference(q[a:a + 128], k[:a + 128], clean[:a + 128], [0, 128], [0, a + 128])
        seen = ~hit[a:a + 128]
        assert ((got[a:a + 128].double() - want).abs() <= tol)[seen].all()


@pytest.mark.gpu
def test_scratch_is_of_the_calls_size():
    """None for up to 128 keys, one round's for a few thousand tokens, all of it for long prompts; never more than what suffices for every call."""
    import crispybits_kernels as ck
    from crispybits_kernels import _C
    lib = _C._lib
    lib.cb_prompt_attention_scratch.argtypes, lib.cb_prompt_attention_scratch.restype = [ctypes.c_int, ctypes.POINTER(ctypes.c_size_t)], ctypes.c_size_t

    def need(tq, tk, h, b, d=128):
        c = ctypes.c_size_t(99)
        return lib.cb_prompt_attention_scratch_for(tq, tk, h, b, d, c), c.value

    c = ctypes.c_size_t(0)
    most = lib.cb_prompt_attention_scratch(128, c), c.value
    assert need(37, 37, 32, 1) == need(128, 128, 64, 5) == need(5, 0, 4, 1) == (0, 0)
    assert need(2000, 2000, 32, 1) == (most[0] // 4, most[1] // 4) and need(16384, 16384, 32, 1) == most
    sizes = [need(1 << a, 1 << b, h, s) for a in (0, 8, 14, 29) for b in (0, 8, 14, 29) for h in (1, 40, (1 << 20) - 1) for s in (1, 9, 1 << 24)]
    assert all(n <= most[0] and k <= most[1] for n, k in sizes)
    x = rand(300, 4, 128, torch.float16, 1)
    s = torch.cuda.Stream()
    _C._attention_eager.pop((torch.cuda.current_device(), s.cuda_stream), None)      # torch hands streams out again
    with torch.cuda.stream(s):
        ck.prompt_attention(x[:100], x[:100], x[:100], i32([0, 37, 100]))
        have = _C._attention_eager[(torch.cuda.current_device(), s.cuda_stream)]
        assert have[1].numel() < 1024
        want = ck.prompt_attention(x, x, x, i32([0, 300]))
        assert _C._attention_eager[(torch.cuda.current_device(), s.cuda_stream)][1].numel() == most[0] // 4
    torch.cuda.synchronize()
    check(want, reference(x, x, x, [0, 300], [0, 300]))


@pytest.mark.gpu
def test_captures_of_many_prompts_leave_counters_for_others():
    """Three captures of forty calls each need twice what was prepared: the eager calls between them, a warm-up's, make up for it."""
    import crispybits_kernels as ck
    from crispybits_kernels import _C
    n = 6000
    x, cu = rand(n, 40, 64, torch.float16, 1), i32([0, n])
    k = x[:, :1].contiguous()
    want = ck.prompt_attention(x, k, k, cu)
    slab, graphs = _C._attention_slab[torch.cuda.current_device()], []
    for _ in range(3):
        assert torch.equal(ck.prompt_attention(x, k, k, cu), want)
        g, before = torch.cuda.CUDAGraph(), slab[1]
        assert before <= slab[0].numel() // 2
        with torch.cuda.graph(g):
            outs = [ck.prompt_attention(x, k, k, cu)]
            for _ in range(39):
                outs = [ck.prompt_attention(x, k, k, cu, out=outs[0])]
        used = slab[1] - before
        assert used > 0
        graphs.append((g, outs))
    for g, outs in graphs * 2:
        g.replay()
        assert torch.equal(outs[0], want)


def test_more_sequences_than_the_walk_can_take_are_refused():
    from crispybits_kernels import _C
    lib, s6 = _C._lib, (ctypes.c_int64 * 6)(*[128] * 6)
    assert lib.cb_prompt_attention(256, 256, 256, s6, 256, 4, 4, 2, 2, 64, 1, 256, 256, (1 << 22) + 1, 1.0, 1, 256, 1 << 20, 256, 1 << 40, 0) == 1
    assert b"sequences" in lib.cb_last_error()


@pytest.mark.gpu
def test_as_many_sequences_as_there_may_be():
    """2^22 sequences, most of them empty: the walk over their bounds stays far inside the others' waits."""
    import crispybits_kernels as ck
    from crispybits_kernels import _C
    B, n = 1 << 22, 700
    q, k, v = rand(n, 2, 64, torch.float16, 1), rand(n, 1, 64, torch.float16, 2), rand(n, 1, 64, torch.float16, 3)
    cu = torch.zeros(B + 1, dtype=torch.int32)
    cu[100:], cu[B // 2:], cu[B:] = 300, 301, n
    _C.decode_status()
    t0, t1 = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    dev = cu.to(DEV)
    t0.record()
    got = ck.prompt_attention(q, k, v, dev)
    t1.record()
    torch.cuda.synchronize()
    assert _C.decode_status() == 0
    print("ms", t0.elapsed_time(t1))
    want = [0, 300, 301, n]
    check(got, reference(q, k, v, want, want))


def rounds(lens, keys, heads, causal):
    """In how many rounds a call goes through its work: by units, key tiles of each tile of 256 queries and three more."""
    units = 0
    for lq, lk in zip(lens, keys):
        for r in range(0, lq, 256):
            seen = [min(lk, r + x + min(lq - r - x, 128) + lk - lq) if causal else lk for x in (0, 128) if lq > r + x]
            units += 3 + max(max(0, -(-n // 128)) for n in seen)
    return min(max(units * heads // (100 * torch.cuda.get_device_properties(0).multi_processor_count), 1), 4)


@pytest.mark.gpu
@pytest.mark.parametrize("lens,past,heads,d,dtype,causal,want", [([8192, 300, 1, 5000], [0] * 4, 24, 64, torch.float16, True, 2),
                                                                ([4000, 0, 8000], [3000, 500, 2000], 24, 128, torch.bfloat16, True, 3),
                                                                ([3000, 2000], [9000, 6000], 48, 64, torch.bfloat16, False, 4),
                                                                ([700] * 60, [1500] * 60, 8, 128, torch.float16, True, 1)])
def test_work_in_several_rounds(lens, past, heads, d, dtype, causal, want):
    """Work of more than two rounds: a CTA comes back for other parts, with scratch and counters of their own.  Some heads against their definition."""
    import crispybits_kernels as ck
    keys = [n + p for n, p in zip(lens, past)]
    if torch.cuda.get_device_properties(0).multi_processor_count == 148:
        assert rounds(lens, keys, heads, causal) == want
    cq, ckv = offsets(lens), offsets(keys)
    q, k, v = rand(cq[-1], heads, d, dtype, 1), rand(ckv[-1], heads // 4, d, dtype, 2), rand(ckv[-1], heads // 4, d, dtype, 3)
    got = ck.prompt_attention(q, k, v, i32(cq), i32(ckv), causal=causal)
    assert torch.equal(got, ck.prompt_attention(q, k, v, i32(cq), i32(ckv), causal=causal))
    for h in (0, 1, heads // 2 - 1, heads // 2, heads - 2, heads - 1):
        check(got[:, h:h + 1], reference(q[:, h:h + 1], k[:, h // 4:h // 4 + 1], v[:, h // 4:h // 4 + 1], cq, ckv, causal=causal))


@pytest.mark.gpu
def test_the_largest_scales():
    """3e38 is finite, and so is what queries of zeros make of it."""
    import crispybits_kernels as ck
    q, k, v = torch.zeros(200, 2, 64, dtype=torch.bfloat16, device=DEV), rand(200, 1, 64, torch.bfloat16, 2), rand(200, 1, 64, torch.bfloat16, 3)
    for scale in (3e38, -3e38):
        check(ck.prompt_attention(q, k, v, i32([0, 200]), scale=scale), reference(q, k, v, [0, 200], [0, 200], 0.0))


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_values_that_are_all_not_finite(bad):
    """A column of v that is not finite throughout: every query sees one, and nothing has to be found out at length."""
    import crispybits_kernels as ck
    n = 4000
    q, k, v = rand(n, 4, 64, torch.float16, 1), rand(n, 2, 64, torch.float16, 2), rand(n, 2, 64, torch.float16, 3)
    want, tol = reference(q, k, v, [0, n], [0, n])
    v[:, 0, 5] = bad
    v[0, 1] = bad
    got = ck.prompt_attention(q, k, v, i32([0, n]))
    hit = torch.zeros(4, 64, dtype=torch.bool, device=DEV)
    hit[:2, 5] = hit[2:] = True
    assert (~torch.isfinite(got) == hit).all() and ((got.double() - want).abs() <= tol)[:, ~hit].all()
