"""Keeping a tree's accepted path in the cache, bit for bit, and a whole speculative step (run with -m gpu on a B200)."""

import numpy as np
import pytest
import torch

from visible_ref import random_tree

pytestmark = pytest.mark.gpu

FP16, BF16, FP32 = torch.float16, torch.bfloat16, torch.float32
KINDS = [(FP16, 0, 16), (BF16, 0, 128), (FP32, 0, 48), (FP16, 8, 128), (FP16, 4, 128), (FP16, 8, 16), (FP16, 4, 8)]


def _random_cache(s, need, hkv, d, page, dtype, bits, seed):
    import easymlx_b200 as emlx

    cache = emlx.PageCacheView.init(num_seqs=s, max_seq_len=need, num_kv_heads=hkv, head_dim=d, block_size=page, dtype=dtype,
                                    cache_dtype=f"affine{bits}" if bits else None)
    g = torch.Generator(device="cuda").manual_seed(seed)
    for t in (cache.key_cache, cache.value_cache, cache.k_scales, cache.k_biases, cache.v_scales, cache.v_biases):
        if t is not None:
            if t.dtype == torch.uint8:
                t.copy_(torch.randint(0, 256, t.shape, generator=g, device="cuda", dtype=torch.uint8))
            else:
                t.copy_(torch.randn(t.shape, generator=g, device="cuda"))
    cache.block_tables.copy_(torch.randperm(cache.block_tables.numel(), generator=g, device="cuda").reshape(cache.block_tables.shape))
    return cache


def _rows(cache):
    """Everything the cache holds per (page, offset) in a form that rows can be moved in, as numpy."""
    nb, bs, h, d = cache.num_blocks, cache.block_size, cache.num_kv_heads, cache.head_dim
    out = [cache.key_cache.view(nb, bs, -1).view(torch.uint8).cpu().numpy()]
    if not cache.is_affine:
        return out + [cache.value_cache.view(nb, bs, -1).view(torch.uint8).cpu().numpy()]
    v = cache.value_cache.cpu().numpy()
    if cache.cache_bits == 4:
        v = np.stack([v & 15, v >> 4], -1).reshape(nb, h, d, bs)
    out.append(np.ascontiguousarray(v.transpose(0, 3, 1, 2)))
    for t in (cache.k_scales, cache.k_biases, cache.v_scales, cache.v_biases):
        out.append(np.ascontiguousarray(t.view(torch.int16).cpu().numpy().transpose(0, 2, 1, 3)))
    return out


def _moved(rows, table, page, ctx, paths):
    rows = [r.copy() for r in rows]
    for s, path in enumerate(paths):
        for r in rows:
            at = lambda p: (table[s, p // page], p % page)
            picked = [r[at(ctx[s] + a)].copy() for a in path]
            for j, x in enumerate(picked):
                r[at(ctx[s] + j)] = x
    return rows


@pytest.mark.parametrize("dtype,bits,page", KINDS)
@pytest.mark.parametrize("host", [False, True])
def test_rows_move_bit_for_bit(dtype, bits, page, host):
    """Paths that chain (a destination is another token's source), that stay where they are, that cross pages, empty ones."""
    ctx = [0, 127, 30, 64, 5]
    paths = [[0, 2, 4, 5, 9], [0, 1, 2], [], [69], list(range(0, 140, 2))]
    slots = [3, 0, 6, 1, 5]
    cache = _random_cache(7, 300, 3, 64, page, dtype, bits, 1)
    for c, x in zip(ctx, slots):
        cache.kv_lens[x] = c
    table = cache.block_tables[slots].cpu().numpy()
    expect = _moved(_rows(cache), table, page, ctx, paths)
    lens = cache.kv_lens.cpu().clone()
    width = max(len(p) for p in paths)
    padded = torch.tensor([p + [-1] * (width - len(p)) for p in paths], dtype=torch.int32)
    got = cache.commit_tree(slots if host else torch.tensor(slots, device="cuda"), paths if host else padded.cuda().long())
    for a, b in zip(_rows(cache), expect):
        assert np.array_equal(a, b)
    assert got.tolist() == [c + len(p) for c, p in zip(ctx, paths)]
    for c, p, x in zip(ctx, paths, slots):
        lens[x] = c + len(p)
    assert torch.equal(cache.kv_lens.cpu(), lens)


@pytest.mark.parametrize("shared", [False, True])
def test_many_layers_in_few_launches(shared):
    """35 layers need two launches; layers that share their lengths advance them once."""
    import easymlx_b200 as emlx
    from easymlx_b200 import _native

    ctx, paths = [10, 33], [[0, 3, 7], [1]]
    views = [_random_cache(2, 64, 2, 64, 16, FP16, 0, i) for i in range(35)]
    for v in views:
        if shared:
            v.kv_lens, v.block_tables = views[0].kv_lens, views[0].block_tables
        v.kv_lens.copy_(torch.tensor(ctx, dtype=torch.int32))
    expect = [_moved(_rows(v), v.block_tables.cpu().numpy(), 16, ctx, paths) for v in views]
    cache = emlx.PageCache(views)
    before = _native.launch_count()
    same = cache.commit_tree([0, 1], paths, advance=False)
    assert _native.launch_count() - before == 2
    assert same.tolist() == [13, 34] and views[3].kv_lens.tolist() == ctx
    for v, e in zip(views, expect):
        assert all(np.array_equal(a, b) for a, b in zip(_rows(v), e))
    emlx.PageTableRunner(views).commit_tree([0, 1], [[0], []])
    assert all(v.kv_lens.tolist() == [11, 33] for v in views)


def test_faulty_paths_leave_their_sequence_alone():
    cache = _random_cache(6, 64, 2, 64, 16, FP16, 0, 5)
    cache.kv_lens.copy_(torch.tensor([5, 5, 5, 60, 5, 5], dtype=torch.int32))
    cache.block_tables[4, 1] = -1
    rows = _rows(cache)
    paths = torch.tensor([[2, 1], [0, 0], [0, 3], [0, 9], [0, 12], [1, 4]], dtype=torch.int32, device="cuda")
    slots = torch.tensor([0, 1, 2, 3, 4, 2], device="cuda")  # slot 2 twice: the first listing counts
    expect = _moved(rows, cache.block_tables[[2]].cpu().numpy(), 16, [5], [[0, 3]])
    with pytest.raises(RuntimeError, match="not increasing"):
        cache.commit_tree(slots, paths)
    assert all(np.array_equal(a, b) for a, b in zip(_rows(cache), expect))
    assert cache.kv_lens.tolist() == [5, 5, 7, 60, 5, 5]
    got = cache.commit_tree([5], [[0, 1]])  # reported once, then clean
    assert got.tolist() == [7]


def test_refusals():
    cache = _random_cache(3, 64, 2, 64, 16, FP16, 0, 6)
    with pytest.raises(ValueError, match="twice"):
        cache.commit_tree([0, 0], [[0], [0]])
    with pytest.raises(IndexError):
        cache.commit_tree([3], [[0]])
    with pytest.raises(ValueError, match="increasing"):
        cache.commit_tree([0], [[1, 1]])
    with pytest.raises(ValueError, match="accepted"):
        cache.commit_tree([0], torch.zeros(2, 3, dtype=torch.int32, device="cuda"))
    assert cache.commit_tree([], []).shape == (0,)
    assert cache.commit_tree([0], [[]]).tolist() == [0]


def _chain(cache, tokens, qkv, rope, meta_args, scale, slot=0):
    """The plain way: append the tokens one after the other and attend with each."""
    import easymlx_b200 as emlx

    outs = []
    perf = emlx.AttentionPerformer(scale=scale)
    for t in tokens:
        q, k, v = (x[t:t + 1] for x in qkv)
        meta = emlx.PageMetadata(query_start_loc=emlx.build_query_start_loc([1]), slot_ids=(slot,), **meta_args)
        outs.append(perf(q, k, v, cache_view=cache, cache_metadata=meta, rope=rope))
    return torch.cat(outs)


@pytest.mark.parametrize("bits", [0, 8])
@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 4)])
def test_speculative_step_equals_plain_decoding(bits, window, sinks):
    """Write a tree, attend with it, keep a path: rows of the path are those that decoding the path token by token gives,
    and so is the cache the next step reads."""
    import easymlx_b200 as emlx
    from easymlx_b200.layers.rotary import RotaryEmbedding

    hq, hkv, d, ctx = 8, 2, 128, 300
    parents = [-1, 0, 0, 1, 1, 2, 3, 5, 5, 7]
    path = [0, 2, 5, 8]
    rope, scale = RotaryEmbedding(d, base=1e6), d ** -0.5
    g = torch.Generator(device="cuda").manual_seed(3)
    make = lambda n, h: torch.randn(n, h, d, generator=g, device="cuda").to(FP16)
    caches = [emlx.PageCacheView.init(num_seqs=1, max_seq_len=512, num_kv_heads=hkv, head_dim=d, block_size=128,
                                      cache_dtype=f"affine{bits}" if bits else None) for _ in range(2)]
    k0, v0 = make(ctx, hkv), make(ctx, hkv)
    for c in caches:
        c.append(0, k0, v0)
    n = len(parents)
    qkv = (make(n, hq), make(n, hkv), make(n, hkv))
    extra = dict(sliding_window=window, sink_tokens=sinks)
    meta = emlx.PageMetadata(query_start_loc=emlx.build_query_start_loc([n]), slot_ids=(0,),
                             tree_mask=emlx.build_tree_mask([parents], device="cuda"), **extra)
    q, kc, vc, resolved = caches[0].concatenate_to_cache(*qkv, cache_metadata=meta, rope=rope, advance=False)
    op = emlx.OperationRegistry.create("unified_attention")
    tree = op(query=q, key=kc, value=vc, cache_metadata=resolved, cache_view=caches[0], scale=scale).attention_outputs
    plain = _chain(caches[1], path, qkv, rope, extra, scale)
    # the same numbers through other kernels and groupings of the keys: a few roundings of fp16 weights and outputs
    assert (tree[path].float() - plain.float()).abs().max() < 4e-3
    assert caches[0].commit_tree([0], [path]).tolist() == [ctx + len(path)]
    pos = ctx + len(path)
    rows = [c.gather_kv_cache(c.block_tables, [0, pos], out_dtype=torch.float32) for c in caches]
    # keys rotated at 64-bit angles on one side, at 32-bit ones on the other: angles up to ~310 differ by 2^-16
    step = 0.05 if bits == 8 else 4e-3
    assert (rows[0][0] - rows[1][0]).abs().max() < step and torch.equal(rows[0][1], rows[1][1])
    nxt = (make(1, hq), make(1, hkv), make(1, hkv))
    a, b = (_chain(c, [0], nxt, rope, extra, scale) for c in caches)
    assert (a.float() - b.float()).abs().max() < 4e-3


def test_captured_step_and_commit():
    """A verify step captured in a graph (write, attention) beside an eager one on the same cache geometry, replayed with new
    inputs; two captured graphs replayed at once on two streams."""
    import easymlx_b200 as emlx
    from easymlx_b200.runtime import AttentionStep

    rng = np.random.default_rng(1)
    steps, expect = [], []
    for i in range(2):
        cache = _random_cache(2, 900, 2, 128, 128, FP16, 0, i)
        cache.kv_lens.copy_(torch.tensor([700, 33], dtype=torch.int32))
        q, k, v = (torch.randn(40, h, 128, device="cuda").half() for h in (8, 2, 2))
        mask = emlx.build_tree_mask([random_tree(rng, 20), random_tree(rng, 20)], device="cuda")
        step = AttentionStep(cache, q, k, v, [20, 20], (0, 1), tree_mask=mask).capture(warmup=1)
        fresh = torch.randn_like(q)
        q.copy_(fresh)
        mask.copy_(emlx.build_tree_mask([random_tree(rng, 20), random_tree(rng, 20)]))
        eager = AttentionStep(cache, q, k, v, [20, 20], (0, 1), tree_mask=mask)
        expect.append(eager.step().clone())
        steps.append(step)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in steps]
    for _ in range(5):
        for step, stream in zip(steps, streams):
            with torch.cuda.stream(stream):
                step.step()
    torch.cuda.synchronize()
    for step, e in zip(steps, expect):
        assert torch.equal(step.out, e)


@pytest.mark.parametrize("bits", [None, 8, 4])
def test_a_tree_and_a_causal_chunk_through_the_performer(bits):
    """One step through the model's entry: a tree, a causal chunk and a finished slot; the tree keeps a path, the chunk all of
    its tokens.  The cache is then that of a step with those tokens only, bit for bit."""
    import easymlx_b200 as emlx

    hq, hkv, d = 8, 2, 64
    g = torch.Generator(device="cuda").manual_seed(5)
    make = lambda n, h: torch.randn(n, h, d, generator=g, device="cuda").to(FP16)
    caches = [emlx.PageCacheView.init(num_seqs=3, max_seq_len=256, num_kv_heads=hkv, head_dim=d, block_size=16,
                                      cache_dtype=f"affine{bits}" if bits else None) for _ in range(2)]
    for slot, ctx in ((2, 37), (0, 16)):
        rows = (make(ctx, hkv), make(ctx, hkv))
        for c in caches:
            c.append(slot, *rows)
    parents, chunk, path = [-1, 0, 0, 1, -1, 4], 21, [0, 2]
    n = len(parents) + chunk
    q, k, v = make(n, hq), make(n, hkv), make(n, hkv)
    mask = torch.zeros(n, 1, dtype=torch.int64, device="cuda")
    mask[: len(parents)] = emlx.build_tree_mask([parents], device="cuda")
    meta = emlx.PageMetadata(query_start_loc=emlx.build_query_start_loc([len(parents), chunk]), slot_ids=(2, 0), tree_mask=mask,
                             tree_seqs=torch.tensor([1, 0], dtype=torch.int32, device="cuda"))
    performer = emlx.AttentionPerformer(scale=d ** -0.5)
    out = performer(q, k, v, cache_view=caches[0], cache_metadata=meta, advance=False)
    assert caches[0].kv_lens.tolist() == [16, 0, 37]
    assert caches[0].commit_tree([2, 0], [path, list(range(chunk))]).tolist() == [39, 37]
    assert caches[0].kv_lens.tolist() == [37, 0, 39]
    keep = torch.tensor(path + list(range(len(parents), n)), device="cuda")
    plain = emlx.PageMetadata(query_start_loc=emlx.build_query_start_loc([len(path), chunk]), slot_ids=(2, 0))
    want = performer(q[keep], k[keep], v[keep], cache_view=caches[1], cache_metadata=plain)
    # the same keys in other groupings: weights and outputs each rounded to fp16, |v| < 5.  Codes: keys may be rounded to fp16 on
    # one side, a score moves by |q| |k| 2^-11 / 8 < 12 * 12 * 2^-14 and the output by twice that of |v|
    bound = 4 * 5 * 2.0 ** -11 + (2 * 5 * 144 * 2.0 ** -14 if bits else 0)
    assert (out[keep].float() - want.float()).abs().max() < bound
    assert torch.equal(caches[0].kv_lens, caches[1].kv_lens)
    for slot in (0, 2):
        lens = [0, int(caches[0].kv_lens[slot])]
        a, b = (c.gather_kv_cache(c.block_tables[slot:slot + 1], lens, out_dtype=torch.float32) for c in caches)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
