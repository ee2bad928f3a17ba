"""The decode stack with attention: prompts into the 4-bit cache, then decode steps over it.

CPU: host code and head sharding (two gloo ranks equal one) with the stand-in backend.  GPU: the operators together, against the
same data flow with the attention computed in 64 bits."""
import os
import socket
import sys

import pytest
import torch

from conftest import PKG, ROOT


@pytest.fixture
def stand_in():
    import attention_backend
    from crispybits_kernels import ops
    prev = ops._C
    ops.set_backend(attention_backend)
    yield attention_backend
    ops.set_backend(prev if prev is not None else "cuda")


def make(rank=0, world=1):
    from crispybits_kernels.stack import DecodeStack, StackCache
    from test_stack import oracle_packer
    st = DecodeStack(2, 256, 512, bitmap=[3, 4], rank=rank, world=world, device="cpu", std=0.05, packer=oracle_packer)
    return st, StackCache(st, 3, 40, head_dim=64, page_size=16)


def run(st, cache):
    """Two pieces of three prompts, then three steps."""
    gen = torch.Generator().manual_seed(0)
    x = [torch.randn(n, 256, generator=gen).half() for n in (8, 14, 3, 3, 3)]
    out = [st.prefill(x[0], [5, 1, 2], cache), st.prefill(x[1], [3, 4, 7], cache, past=[5, 1, 2])]
    return out + [st.step(t, cache=cache) for t in x[2:]]


def test_pieces_and_steps_equal_one_prompt(stand_in):
    """What the last step answers does not depend on how its sequence came into the cache (but for pieces of a prompt,
    which see their own keys in 4 bits)."""
    st, cache = make()
    out = run(st, cache)
    assert cache.lengths.tolist() == [11, 8, 12] and [o.shape for o in out] == [(8, 256), (14, 256)] + [(3, 256)] * 3
    gen = torch.Generator().manual_seed(0)
    x = [torch.randn(n, 256, generator=gen).half() for n in (8, 14, 3, 3, 3)]
    st2, cache2 = make()
    a, b = x[0].split([5, 1, 2]), x[1].split([3, 4, 7])
    st2.prefill(torch.cat([torch.cat((a[i], b[i])) for i in range(3)]), [8, 5, 9], cache2)
    for t in x[2:]:
        y = st2.step(t, cache=cache2)
    # Keys of a row may round another way in a product of other rows, and a 4-bit code then differs by a step: 1/15 of a group's range
    # (about 5 of its standard deviations) in one of at least 8 tokens' keys or values, less than 1/20 of an output's size.
    size = out[4].float().abs().max()
    assert (y.float() - out[4].float()).abs().max() <= size / 20
    assert (out[4].float() - st.step(x[4]).float()).abs().max() > size / 5       # the plain step passes Q on
    with pytest.raises(ValueError):
        st.step(x[4][:2], cache=cache)
    with pytest.raises(ValueError):
        st.prefill(x[0], [5, 1, 1], cache)
    other, _ = make()
    other.n_blocks = 1
    with pytest.raises(ValueError):
        other.step(x[4], cache=cache)


def test_a_backend_without_attention_is_refused():
    import oracle_backend
    from crispybits_kernels import KV4Cache, ops
    prev = ops._C
    ops.set_backend(oracle_backend)
    try:
        with pytest.raises(RuntimeError):
            KV4Cache.empty(1, 1, 64, device="cpu")
    finally:
        ops.set_backend(prev if prev is not None else "cuda")


def _worker(rank, world, port, out_path):
    sys.path[:0] = [ROOT, PKG, os.path.join(ROOT, "tests")]
    import torch.distributed as dist

    import attention_backend
    from crispybits_kernels import ops
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    ops.set_backend(attention_backend)
    out = run(*make(rank, world))
    if rank == 0:
        torch.save({"sharded": out, "full": run(*make())}, out_path)
    dist.barrier()
    dist.destroy_process_group()


def test_two_ranks_with_half_the_heads_each_match_one(tmp_path):
    import torch.multiprocessing as mp
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    mp.spawn(_worker, args=(2, port, str(tmp_path / "res.pt")), nprocs=2, join=True)
    res = torch.load(tmp_path / "res.pt")
    for a, b in zip(res["sharded"], res["full"]):
        assert (a.float() - b.float()).abs().max() <= 2e-3 * b.float().abs().max()


# ------------------------------------------------------------------------------------------------ GPU
@pytest.mark.gpu
@pytest.mark.parametrize("head_dim", [64, 128])
def test_stack_with_attention_on_gpu(head_dim):
    """Prompt, a second piece, steps (eager, then captured and replayed): every output against the same linears with the attention
    in 64 bits over the values the cache has to hold."""
    import crispybits_kernels as ck
    from crispybits_kernels import ops
    from crispybits_kernels.stack import DecodeStack, StackCache
    from test_kv4 import quantise64, values64
    ops.set_backend("cuda")
    st = DecodeStack(2, 512, 1024, bitmap=[4, 3], device="cuda", std=0.05)
    cache = StackCache(st, 3, 200, head_dim=head_dim, page_size=32)
    heads = 512 // head_dim
    gen = torch.Generator().manual_seed(1)
    rows = lambda n: torch.randn(n, 512, generator=gen).half().cuda()
    past = [[torch.empty(0, 2, heads, head_dim, device="cuda", dtype=torch.half) for _ in range(3)] for _ in st.blocks]
    held = lambda t: values64(*quantise64(t, 64)).to(torch.half).double()

    def attend(q, kv, quantised):
        k, v = (held(t) if quantised else t.double() for t in kv.unbind(1))
        n, t = k.shape[0], q.shape[0]
        s = torch.einsum("thd,nhd->htn", q.double(), k) * head_dim ** -0.5
        s = s.masked_fill(torch.arange(n, device="cuda")[None] > torch.arange(t, device="cuda")[:, None] + n - t, float("-inf"))
        return torch.einsum("htn,nhd->thd", torch.softmax(s, -1), v).half()

    def expected(x, lens, step, quantised):
        kw = dict(decode_threshold=8) if step else {}
        y = None
        for i, blk in enumerate(st.blocks):
            q, k, v = (t.view(-1, heads, head_dim) for t in ck.fused_qkv(x, blk.q, blk.k, blk.v, **kw))
            parts, at = [], 0
            for s, n in enumerate(lens):
                past[i][s] = torch.cat((past[i][s], torch.stack((k[at:at + n], v[at:at + n]), 1)))
                parts.append(attend(q[at:at + n], past[i][s], quantised))
                at += n
            a = ck.packed_linear(torch.cat(parts).flatten(1), blk.o, **kw)
            y = ck.packed_linear(ck.fused_gate_up(a, blk.gate, blk.up, **kw), blk.down, **kw)
        return y

    def close(got, want):
        # an output of the attention is off by a few 2^-11 of the values' size at most; the three linears behind it carry that on
        assert (got.float() - want.float()).abs().max() <= 6e-3 * want.float().abs().max()

    x = rows(70 + 3 + 20)
    close(st.prefill(x, [70, 3, 20], cache), expected(x, [70, 3, 20], False, False))
    x = rows(10 + 40 + 1)
    close(st.prefill(x, [10, 40, 1], cache, past=[70, 3, 20]), expected(x, [10, 40, 1], False, True))
    for _ in range(3):
        x = rows(3)
        close(st.step(x, cache=cache), expected(x, [1, 1, 1], True, True))
    assert cache.lengths.tolist() == [83, 46, 24]
    x, graph = rows(3), torch.cuda.CUDAGraph()
    before = cache.lengths.clone()
    st.step(x, cache=cache)                                    # warm up, undone
    cache.lengths.copy_(before)
    with torch.cuda.graph(graph):
        y = st.step(x, cache=cache)
    for _ in range(3):
        x.copy_(rows(3))
        graph.replay()
        close(y, expected(x, [1, 1, 1], True, True))
    assert cache.lengths.tolist() == [86, 49, 27]
    from crispybits_kernels import _C
    assert _C.decode_status() == 0


def test_append_refuses_batches_that_do_not_fit_the_page_table(stand_in):
    """A batch of another number of sequences, or k and v of different [B, T], would put tokens into sequences that are not theirs."""
    from crispybits_kernels import KV4Cache, kv4_append, kv4_read
    cache = KV4Cache.empty(4, 2, 64, 16, device="cpu")
    table, starts = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    x = torch.randn(8, 2, 64).half()
    for k, v in ((x.view(4, 2, 2, 64), x.view(4, 2, 2, 64)), (x.view(1, 8, 2, 64), x.view(1, 8, 2, 64)), (x.view(2, 4, 2, 64), x.view(4, 2, 2, 64)),
                 (x.view(2, 4, 2, 64), x), (x, x.view(2, 4, 2, 64)), (x[:7], x[:7])):
        with pytest.raises(ValueError):
            kv4_append(cache, k, v, table, starts)
    kv4_append(cache, x.view(2, 4, 2, 64), x.view(2, 4, 2, 64), table, starts)
    a = kv4_read(cache, table, starts, None, 8)
    kv4_append(cache, x, x, table, starts)                         # packed, as many tokens of each
    assert torch.equal(a[0], kv4_read(cache, table, starts, None, 8)[0])


def test_a_past_that_is_not_the_caches_and_tokens_without_room_are_refused(stand_in):
    """Nothing is appended by a call that is refused."""
    st, cache = make()
    assert cache.capacity == 48                                    # 40 tokens in pages of 16
    x = lambda n: torch.randn(n, 256, generator=torch.Generator().manual_seed(n)).half()
    st.prefill(x(8), [5, 1, 2], cache)
    for lens, past in (([5, 1, 2], None), ([5, 1, 2], [5, 1, 3]), ([5, 1, 2], [5, 1]), ([5, 1, 2], [0, 0, 0]), ([44, 0, 0], [5, 1, 2]), ([-1, 1, 1], [5, 1, 2])):
        with pytest.raises(ValueError):
            st.prefill(x(sum(lens)), lens, cache, past=past)
        assert cache.lengths.tolist() == [5, 1, 2]
    st.prefill(x(41), [41, 0, 0], cache, past=[5, 1, 2])
    for n in (47, 48):
        st.step(x(3), cache=cache)
        assert cache.lengths.tolist()[0] == n
    with pytest.raises(ValueError):
        st.step(x(3), cache=cache)
    assert cache.lengths.tolist() == [48, 3, 4]
    cache.lengths.copy_(torch.tensor([47, 0, 1]))                  # sequences start again: the lengths are theirs who own the cache
    st.step(x(3), cache=cache)
    with pytest.raises(ValueError):
        st.step(x(3), cache=cache)
    cache.lengths.zero_()
    st.prefill(x(8), [5, 1, 2], cache)
    assert cache.lengths.tolist() == [5, 1, 2]


def test_a_cache_made_in_inference_mode(stand_in):
    with torch.inference_mode():
        from crispybits_kernels.stack import StackCache
        st = make()[0]
        cache = StackCache(st, 3, 16, head_dim=64, page_size=16)
        x = torch.randn(3, 256, generator=torch.Generator().manual_seed(1)).half()
        st.prefill(x.repeat(16, 1), [16, 16, 16], cache)
        cache.lengths.fill_(15)
        st.step(x, cache=cache)
        with pytest.raises(ValueError):
            st.step(x, cache=cache)


@pytest.mark.gpu
def test_replays_of_a_captured_step_count_for_the_eager_ones():
    import crispybits_kernels as ck
    from crispybits_kernels import ops
    from crispybits_kernels.stack import DecodeStack, StackCache
    ops.set_backend("cuda")
    st = DecodeStack(1, 256, 512, bitmap=[4], device="cuda", std=0.05)
    cache = StackCache(st, 2, 16, head_dim=64, page_size=16)
    x, graph = torch.randn(2, 256, device="cuda").half(), torch.cuda.CUDAGraph()
    st.step(x, cache=cache)
    with torch.cuda.graph(graph):
        st.step(x, cache=cache)
    for _ in range(14):
        graph.replay()
    st.step(x, cache=cache)
    assert cache.lengths.tolist() == [16, 16]
    with pytest.raises(ValueError):
        st.step(x, cache=cache)
    graph.replay()                                                 # left out, and said so
    from crispybits_kernels import _C
    assert _C.decode_status() == 3001 and ck.kv4_read(cache.layers[0], cache.page_table, torch.zeros_like(cache.lengths), None, 32)[0].shape[0] == 32
