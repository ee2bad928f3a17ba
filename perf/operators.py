"""The attention operators of the packed decode path, as cases to measure: what each call takes, its plain form in
elementary torch operations, its definition in 64 bits, and the bytes and operations it cannot do without.

Four operators: `prompt_attention` (attention of packed prompts of different lengths over their own keys), and a paged
key/value cache held in 4 bits with `kv4_append` (quantise new tokens into it), `kv4_read` (their values back) and
`kv4_attention` (attention of the newest tokens over it).

The 4-bit format.  The D values of one token and head are cut into groups of `group`; a group keeps lo = its smallest
value and scale = round_T((max - lo) / 15) in the cache's 16-bit type T and one 4-bit code for each value,
    code = round_half_even((x - lo) / scale), at most 15 (0 where scale is 0),      value = code * scale + lo.
"""
import math

import torch

own = False

_DT = {"fp16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one new token of one conversation, 32 heads as in the 7B decode stack: nothing but latency
        {"name": "append_step", "op": "append", "lens": "1", "starts": "1000", "kv_heads": 32, "head_dim": 128,
         "group": 128, "page": 64, "dtype": "fp16"},
        # the keys and values of a batch of prompts of uneven lengths enter the cache at once
        {"name": "append_prompts", "op": "append", "lens": "4096,1,777,2048,33,5000,129,1500", "starts": "0",
         "kv_heads": 32, "head_dim": 128, "group": 64, "page": 64, "dtype": "fp16"},
        # a short history is read back before a prompt goes on
        {"name": "read_short", "op": "read", "lens": "300,45", "starts": "0,7", "kv_heads": 8, "head_dim": 128,
         "group": 64, "page": 16, "dtype": "bf16"},
        # long histories of several conversations are read back, grouped heads
        {"name": "read_long", "op": "read", "lens": "16000,8191,1,30001", "starts": "0,64,5,1", "kv_heads": 8,
         "head_dim": 128, "group": 64, "page": 64, "dtype": "bf16"},
        # one conversation of the 7B stack early on: a launch that is mostly latency
        {"name": "decode_single", "op": "decode", "lens": "777", "new": 1, "heads": 32, "kv_heads": 32,
         "head_dim": 128, "group": 128, "page": 64, "dtype": "fp16"},
        # a serving batch with grouped heads: lengths from none to long, most of them short
        {"name": "decode_batch", "op": "decode",
         "lens": "8192,4097,1,0,2500,700,63,64,65,5000,1023,1300,90,6000,3333,15,2048,480,1800,7100,250,1111,2222,900",
         "new": 1, "heads": 32, "kv_heads": 8, "head_dim": 128, "group": 64, "page": 64, "dtype": "bf16"},
        # one long document, eight query heads to a key head
        {"name": "decode_long", "op": "decode", "lens": "131071", "new": 1, "heads": 64, "kv_heads": 8,
         "head_dim": 128, "group": 64, "page": 64, "dtype": "bf16"},
        # four drafted tokens of each conversation are checked at once, small heads, small pages and groups
        {"name": "decode_draft", "op": "decode", "lens": "2000,1999,3,1024,511,777,1600,40,1290,64,2,900",
         "new": 4, "heads": 12, "kv_heads": 12, "head_dim": 64, "group": 32, "page": 16, "dtype": "fp16"},
        # one short question
        {"name": "prompt_short", "op": "prompt", "lens": "37", "past": "0", "heads": 32, "kv_heads": 32,
         "head_dim": 128, "causal": True, "dtype": "fp16"},
        # prompts of a serving batch, packed, grouped heads
        {"name": "prompt_packed", "op": "prompt", "lens": "4096,1,777,2048,33,128,129,1500,255,1000,600,2000",
         "past": "0", "heads": 32, "kv_heads": 8, "head_dim": 128, "causal": True, "dtype": "bf16"},
        # pieces of long prompts, each attending to what came before it as well; small heads
        {"name": "prompt_pieces", "op": "prompt", "lens": "512,512,300,511", "past": "8192,1536,0,4001", "heads": 12,
         "kv_heads": 12, "head_dim": 64, "causal": True, "dtype": "fp16"},
        # one long document
        {"name": "prompt_long", "op": "prompt", "lens": "16384", "past": "0", "heads": 32, "kv_heads": 32,
         "head_dim": 128, "causal": True, "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "read", "decode", "decode", "prompt", "prompt"])
    head_dim = rng.choice([64, 128])
    case = {"op": op, "head_dim": head_dim, "dtype": rng.choice(["fp16", "bf16"])}
    if op == "prompt":
        kv = rng.choice([1, 2, 3, 4, 8, 12, 16])
        heads = kv * rng.choice([1, 1, 2, 4, 5, 8])
        heads, kv = (heads, kv) if heads <= 32 else (kv, kv)
        lens, past, budget = [], [], 6.0e7           # query-key pairs, well below the longest prompt's
        for _ in range(rng.choice([1, 1, 2, 3, 6, 12])):
            n = _log_int(rng, 1, 6000)
            p = rng.choice([0, 0, 0, _log_int(rng, 1, 8000)])
            if n * (n + p) <= budget:
                budget -= n * (n + p)
                lens.append(n)
                past.append(p)
        if not lens:
            lens, past = [500], [0]
        case.update(lens=",".join(map(str, lens)), past=",".join(map(str, past)), heads=heads, kv_heads=kv,
                    causal=rng.random() < 0.8)
        return case
    kv = rng.choice([1, 2, 3, 4, 5, 8, 12, 32])
    budget = 130000 * 8 // kv * (128 // head_dim)     # tokens in the cache, at most the long document's
    lens = []
    for _ in range(rng.choice([1, 1, 2, 5, 16, 48])):
        n = _log_int(rng, 1, 30000)
        if n <= budget and (op != "append" or sum(lens) + n <= 17000):
            budget -= n
            lens.append(n)
    lens = lens or [100]
    case.update(kv_heads=kv, group=rng.choice([g for g in (32, 64, 128) if g <= head_dim]), page=rng.choice([16, 32, 64]))
    if op == "decode":
        if rng.random() < 0.2:
            lens.append(0)
        case.update(new=rng.choice([1, 1, 1, 2, 3, 4, 7]), heads=kv * rng.choice([1, 2, 3, 4, 8, 16]))
    else:
        case["starts"] = ",".join(str(rng.choice([0, 0, _log_int(rng, 1, 500)])) for _ in lens)
        if op == "append" and rng.random() < 0.4:     # a decode step: one token of each conversation
            lens = [1] * len(lens)
    case["lens"] = ",".join(map(str, lens))
    return case


def _ints(text, count=None):
    v = [int(t) for t in text.split(",")]
    return v * count if count is not None and len(v) == 1 else v


def _shape(case):
    lens = _ints(case["lens"])
    return lens, _ints(case["past"] if case["op"] == "prompt" else case.get("starts", "0"), len(lens))


# ---------------------------------------------------------------------------------------------------- inputs
def _keys(gen, n, heads, d, dtype):
    """Keys as models make them: a few channels are much larger than the others."""
    x = torch.randn(n, heads, d, generator=gen, device="cuda")
    channel = torch.rand(heads, d, generator=gen, device="cuda")
    return (x * (0.5 + channel + 4.0 * (channel > 0.97))).to(dtype)


def _inputs(case, seed):
    """Queries, keys and values (packed over the sequences), from the seed alone."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    lens, past = _shape(case)
    dt, d, kv = _DT[case["dtype"]], case["head_dim"], case["kv_heads"]
    n_keys = sum(lens) + (sum(past) if case["op"] == "prompt" else 0)
    x = {"k": _keys(gen, n_keys, kv, d, dt), "v": torch.randn(n_keys, kv, d, generator=gen, device="cuda").to(dt)}
    if case["op"] == "prompt":
        x["q"] = torch.randn(sum(lens), case["heads"], d, generator=gen, device="cuda").to(dt)
    if case["op"] == "decode":
        x["q"] = torch.randn(len(lens), case["new"], case["heads"], d, generator=gen, device="cuda").to(dt)
    return x, gen


def _offsets(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


# ---------------------------------------------------------------------------------------------------- state
def prepare(case, seed):
    x, gen = _inputs(case, seed)
    lens, second = _shape(case)
    state = dict(x, case=case, lens=lens, second=second, at=_offsets(lens))
    if case["op"] == "prompt":
        state["key_at"] = _offsets([n + p for n, p in zip(lens, second)])
        if own:
            state["ck"] = _package()
            state["cu"], state["cu_k"] = _i32(state["at"]), _i32(state["key_at"])
        return state
    starts = [0] * len(lens) if case["op"] == "decode" else second
    if own:
        ck = state["ck"] = _package()
        page = case["page"]
        need = [max(1, -(-(s + n) // page)) for s, n in zip(starts, lens)]
        cache = state["cache"] = ck.KV4Cache.empty(sum(need) + 1, case["kv_heads"], case["head_dim"], page, case["group"],
                                                   _DT[case["dtype"]], "cuda")
        ids = torch.randperm(sum(need) + 1, generator=gen, device="cuda", dtype=torch.int32)    # pages in any order
        table = torch.zeros(len(lens), max(need), dtype=torch.int32, device="cuda")
        for b, first in enumerate(_offsets(need)[:-1]):
            table[b, :need[b]] = ids[first:first + need[b]]
        state.update(table=table, starts=_i32(starts), lengths=_i32(lens), cu=_i32(state["at"]))
        if case["op"] != "append":
            ck.kv4_append(cache, state["k"], state["v"], table, state["starts"], state["cu"])
            del state["k"], state["v"]
        return state
    if case["op"] != "append":       # what a cache holds: codes, scales and smallest values
        state["k"], state["v"] = (_quantise(state[n], case["group"]) for n in "kv")
    return state


def _package():
    import os
    import sys
    folder = os.path.join(os.getcwd(), "llm_quantization-kernel_b200")
    if folder not in sys.path:
        sys.path.insert(0, folder)
    import crispybits_kernels
    return crispybits_kernels


# ---------------------------------------------------------------------------------------------------- one pass
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    ck, op = s["ck"], s["case"]["op"]
    if op == "prompt":
        return ck.prompt_attention(s["q"], s["k"], s["v"], s["cu"], cu_seqlens_k=s["cu_k"], causal=s["case"]["causal"])
    if op == "decode":
        return ck.kv4_attention(s["q"], s["cache"], s["table"], s["lengths"])
    if op == "append":       # and the values that the new tokens' codes stand for
        ck.kv4_append(s["cache"], s["k"], s["v"], s["table"], s["starts"], s["cu"])
    return ck.kv4_read(s["cache"], s["table"], s["starts"], s["cu"], s["at"][-1])


def _quantise(x, group):
    """In 64 bits: a quotient beside a half would round the other way in 32."""
    g = x.double().unflatten(-1, (-1, group))
    lo = g.amin(-1, keepdim=True)
    scale = ((g.amax(-1, keepdim=True) - lo) / 15).to(x.dtype)
    code = torch.round((g - lo) / torch.where(scale == 0, 1, scale).double()).clamp(0, 15)
    return torch.where(scale == 0, 0, code).to(torch.uint8), scale, lo.to(x.dtype)


def _values(codes, scale, lo):
    return (codes.float() * scale.float() + lo.float()).flatten(-2)


def _plain_attention(q, k, v, first, causal=True):
    """softmax(q k^T / sqrt(d)) v for one sequence: q [t, H, d], k and v [n, Hkv, d] in 32 bits; query j sees the keys up
    to first + j.  Rows of queries in pieces, so that the scores of a long prompt fit."""
    t, heads, d = q.shape
    n, kv = k.shape[:2]
    out = torch.zeros(t, heads, d, device=q.device)
    if n == 0:
        return out
    kt, vt = k.permute(1, 2, 0), v.permute(1, 0, 2)                      # [Hkv, d, n], [Hkv, n, d]
    pos = torch.arange(n, device=q.device)
    piece = max(1, (1 << 29) // max(1, heads * n))
    for a in range(0, t, piece):
        qa = q[a:a + piece].float()
        m = qa.shape[0]
        rows = qa.view(m, kv, heads // kv, d).permute(1, 2, 0, 3).reshape(kv, -1, d)
        sc = ((rows @ kt) / math.sqrt(d)).view(kv, heads // kv, m, n)
        if causal:
            seen = pos[None, :] <= (torch.arange(a, a + m, device=q.device) + first)[:, None]
            sc = sc.masked_fill(~seen, float("-inf"))
        top = sc.amax(-1, keepdim=True)
        p = torch.exp(sc - torch.where(top == float("-inf"), 0.0, top))
        total = p.sum(-1, keepdim=True)
        o = (p.view(kv, -1, n) @ vt).view(kv, heads // kv, m, d) / torch.where(total == 0, 1.0, total)
        out[a:a + m] = o.permute(2, 0, 1, 3).reshape(m, heads, d)
    return out


def _run_plain(s):
    case, op = s["case"], s["case"]["op"]
    dt = _DT[case["dtype"]]
    if op == "append":
        return tuple(_values(*_quantise(s[n], case["group"])).to(dt) for n in "kv")
    if op == "read":
        return tuple(_values(*s[n]).to(dt) for n in "kv")
    if op == "decode":
        out = torch.empty(s["q"].shape, device="cuda")
        for b, n in enumerate(s["lens"]):
            k, v = (_values(*(part[s["at"][b]:s["at"][b + 1]] for part in s[name])) for name in "kv")
            out[b] = _plain_attention(s["q"][b], k, v, n - case["new"])
        return out.to(dt)
    out = torch.empty(s["q"].shape, device="cuda")
    for b in range(len(s["lens"])):
        rows, keys = slice(s["at"][b], s["at"][b + 1]), slice(s["key_at"][b], s["key_at"][b + 1])
        out[rows] = _plain_attention(s["q"][rows], s["k"][keys].float(), s["v"][keys].float(), s["second"][b], case["causal"])
    return out.to(dt)


# ---------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    """From the definition, head by head, in 64 bits."""
    x, _ = _inputs(case, seed)
    lens, second = _shape(case)
    dt = _DT[case["dtype"]]

    def held(name):          # what the cache makes of the values
        y = x[name].double()
        back = torch.empty_like(y)
        for c in range(0, case["head_dim"], case["group"]):
            part = y[..., c:c + case["group"]]
            low, high = part.min(dim=-1, keepdim=True).values, part.max(dim=-1, keepdim=True).values
            step = ((high - low) / 15.0).to(dt).double()
            code = ((part - low) / step).round().clamp(max=15.0).nan_to_num(0.0)
            back[..., c:c + case["group"]] = low + step * code
        return back

    if case["op"] in ("append", "read"):
        return held("k"), held("v")
    k, v = (held("k"), held("v")) if case["op"] == "decode" else (x["k"].double(), x["v"].double())
    q = x["q"].double().flatten(0, -3)
    new = [case["new"]] * len(lens) if case["op"] == "decode" else lens
    keys = lens if case["op"] == "decode" else [n + p for n, p in zip(lens, second)]
    share = case["heads"] // case["kv_heads"]
    out = torch.zeros_like(q)
    row, key = 0, 0
    for t, n in zip(new, keys):
        for h in range(case["heads"] if n else 0):
            kh, vh = k[key:key + n, h // share], v[key:key + n, h // share]
            for a in range(0, t, 4096):
                e = min(t, a + 4096)
                w = torch.einsum("td,nd->tn", q[row + a:row + e, h], kh) * case["head_dim"] ** -0.5
                if case.get("causal", True):
                    last = torch.arange(a, e, device="cuda") + (n - t)
                    w[torch.arange(n, device="cuda")[None] > last[:, None]] = -math.inf
                out[row + a:row + e, h] = torch.softmax(w, -1).nan_to_num(0.0) @ vh
        row, key = row + t, key + n
    return out.view(x["q"].shape)


# ---------------------------------------------------------------------------------------------------- bounds
def work(case):
    lens, second = _shape(case)
    d, kv, op = case["head_dim"], case["kv_heads"], case["op"]
    if op == "prompt":
        pairs = sum(n * (n + p) - (n * (n - 1) // 2 if case["causal"] else 0) for n, p in zip(lens, second))
        size = 2 * d * (2 * sum(lens) * case["heads"] + 2 * (sum(lens) + sum(second)) * kv)
        return {"bytes": size, "flops": 4 * d * case["heads"] * pairs}
    record = 2 * kv * (d // 2 + 4 * (d // case["group"]))          # one token's keys and values in the cache
    tokens = sum(lens)
    if op == "decode":
        rows = len(lens) * case["new"] * case["heads"]
        pairs = case["heads"] * sum(sum(max(0, n - j) for j in range(case["new"])) for n in lens)
        return {"bytes": record * tokens + 2 * 2 * d * rows, "flops": 4 * d * pairs}
    values = 2 * 2 * d * kv * tokens
    if op == "read":
        return {"bytes": record * tokens + values, "flops": 4 * d * kv * tokens}
    return {"bytes": 2 * values + 2 * record * tokens, "flops": 12 * d * kv * tokens}
