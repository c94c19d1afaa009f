"""Cache writes and rotations at given positions against 64-bit angles (run with -m gpu on a B200)."""

import numpy as np
import pytest
import torch

from oracle import kv_quant
from visible_ref import HALF_STEP, random_tree, rotate

pytestmark = pytest.mark.gpu

FP16, BF16, FP32 = torch.float16, torch.bfloat16, torch.float32


def _rope(d, dims=None, axes=3, interleaved=False, **kw):
    from easymlx_b200.layers.rotary import MultiAxisRotaryEmbedding

    dims = dims or d
    half = dims // 2
    if interleaved:
        sections = [half - (axes - 1) * (half // (axes + 1))] + [half // (axes + 1)] * (axes - 1)
    else:
        sections = [half - (axes - 1) * (half // axes)] + [half // axes] * (axes - 1)
    return MultiAxisRotaryEmbedding(dims, base=1e6, sections=sections, interleaved=interleaved, **kw)


def _expected(rope, x, positions):
    pos = np.asarray(positions)
    axis = rope._axis_of_pair.astype(int) if pos.shape[0] > 1 else np.zeros(rope.dims // 2, int)
    return rotate(x.double().numpy(), pos, rope.freqs, axis, rope.dims, rope.scale, rope.traditional, rope.mscale)


def _bound(x, expect, dtype, mscale=1.0):
    """One rounding to the type; cosine and sine are off by at most 2^-22 (the reduced angle, below pi, rounded to 32 bits:
    2^-23, and two units of the function), four 32-bit roundings of products of elements of the row."""
    big = np.abs(x.double().numpy()).max(-1, keepdims=True) * abs(mscale)
    return HALF_STEP[dtype] * np.abs(expect) * 1.01 + 2 * big * (2.0 ** -22 + 3 * 2.0 ** -24) + (6e-8 if dtype == FP16 else 1e-37)


@pytest.mark.parametrize("dtype", [FP16, BF16, FP32])
@pytest.mark.parametrize("d,dims,axes,interleaved,traditional", [
    (128, None, 3, False, False), (128, None, 3, True, False), (64, None, 2, False, False), (256, None, 4, True, False),
    (96, None, 3, False, False), (128, 64, 3, False, False), (64, None, 3, False, True), (80, 34, 1, False, False)])
@pytest.mark.parametrize("t", [1, 5, 700])
def test_rotation_of_a_tensor(dtype, d, dims, axes, interleaved, traditional, t):
    rng = np.random.default_rng(d + t)
    rope = _rope(d, dims, axes, interleaved, traditional=traditional, scale=0.5, mscale=1.25)
    x = torch.from_numpy(rng.standard_normal((t, 3, d)).astype(np.float32)).to(dtype)
    pos = rng.integers(0, 300000, (axes, t)).astype(np.int32)
    got = rope(x.cuda(), offset=torch.from_numpy(pos).cuda())
    expect = _expected(rope, x, pos)
    assert (np.abs(got.double().cpu().numpy() - expect) <= _bound(x, expect, dtype, 1.25)).all()


def test_far_and_negative_positions():
    rope = _rope(128)
    x = torch.ones(4, 1, 128, dtype=FP32)
    pos = np.array([[0, -3, 2 ** 31 - 1, 10 ** 6]] * 3, np.int32)
    expect = _expected(rope, x, pos)
    got = rope(x.cuda(), offset=torch.from_numpy(pos).cuda()).double().cpu().numpy()
    # 2^31 radians leave 53 - 31 bits behind the point in a 64-bit product: 2^-22 of an angle, in either computation
    assert (np.abs(got - expect) <= _bound(x, expect, FP32) + 2 * 2.0 ** -21).all()


def _cache(ctx, qlens, hkv, d, page, dtype, bits, slots, seed=0):
    import easymlx_b200 as emlx

    need = max(ctx) + max(qlens) + 1
    cache = emlx.PageCacheView.init(num_seqs=max(slots) + 1, max_seq_len=need, num_kv_heads=hkv, head_dim=d, block_size=page, dtype=dtype,
                                    cache_dtype=f"affine{bits}" if bits else None)
    g = torch.Generator().manual_seed(seed)
    n = cache.block_tables.numel()
    cache.block_tables.copy_(torch.randperm(n, generator=g).reshape(cache.block_tables.shape))
    lens = torch.zeros(max(slots) + 1, dtype=torch.int32)
    lens[list(slots)] = torch.tensor(ctx, dtype=torch.int32)
    cache.kv_lens.copy_(lens)
    return cache


def _written(cache, slots, ctx, qlens):
    """K and V rows of the step as the cache holds them, ``[T, Hkv, D]`` float64."""
    bt = cache.block_tables[list(slots)].cpu().numpy()
    k, v = cache.dequantize_kv_cache(cache.key_cache, cache.value_cache, out_dtype=torch.float32)
    k, v = k.double().cpu().numpy(), v.double().cpu().numpy()
    at = [(bt[s, p // cache.block_size], p % cache.block_size) for s in range(len(slots)) for p in range(ctx[s], ctx[s] + qlens[s])]
    idx = tuple(np.array(at).T)
    return k[idx], v[idx]


CASES = [(8, 2, 128, 128, FP16, 0), (4, 4, 64, 16, BF16, 0), (6, 1, 128, 64, FP32, 0), (4, 2, 128, 128, FP16, 8), (4, 2, 64, 128, BF16, 4),
         (2, 1, 96, 48, FP16, 0), (2, 2, 256, 32, BF16, 0)]


@pytest.mark.parametrize("hq,hkv,d,page,dtype,bits", CASES)
@pytest.mark.parametrize("qlens", [[1, 1, 1], [5, 0, 130], [1], [400, 700, 900, 500]])
@pytest.mark.parametrize("mode", ["axes", "one", "tree", "slot"])
def test_step_writes_rotated_rows(hq, hkv, d, page, dtype, bits, qlens, mode):
    import easymlx_b200 as emlx

    rng = np.random.default_rng(d + sum(qlens))
    s, t = len(qlens), sum(qlens)
    ctx, slots = [int(x) for x in rng.integers(0, 300, s)], [int(x) for x in rng.permutation(s + 2)[:s]]
    cache = _cache(ctx, qlens, hkv, d, page, dtype, bits, slots)
    rope = _rope(d, interleaved=s == 1)
    q, k, v = (torch.from_numpy(rng.standard_normal((t, h, d)).astype(np.float32)).to(dtype) for h in (hq, hkv, hkv))
    slot_pos = np.concatenate([c + np.arange(n) for c, n in zip(ctx, qlens)]).astype(np.int32)
    more, pos = {}, slot_pos[None]
    if mode == "axes":
        pos = rng.integers(0, 100000, (3, t)).astype(np.int32)
        more["rope_positions"] = torch.from_numpy(pos).cuda()
    elif mode == "one":
        pos = rng.integers(0, 100000, (1, t)).astype(np.int32)
        more["rope_positions"] = torch.from_numpy(pos[0]).cuda().long()
    elif mode == "tree":
        trees = [random_tree(rng, n) for n in qlens]
        more["tree_mask"] = emlx.build_tree_mask(trees, device="cuda")
        depth = []
        for tree in trees:
            level = []
            for p in tree:
                level.append(level[p] + 1 if p >= 0 else 0)
            depth.append(level)
        pos = np.concatenate([c + np.array(x, np.int64) for c, x in zip(ctx, depth)]).astype(np.int32)[None]
    else:
        more.update(sink_tokens=3, sliding_window=50)
    meta = emlx.PageMetadata(query_start_loc=emlx.build_query_start_loc(qlens), slot_ids=tuple(slots), **more)
    before = (cache.key_cache.clone(), cache.value_cache.clone(), cache.kv_lens.clone())
    rotated, kc, vc, resolved = cache.concatenate_to_cache(q.cuda(), k.cuda(), v.cuda(), cache_metadata=meta, rope=rope, query_lens=qlens)
    expect_q, expect_k = _expected(rope, q, pos), _expected(rope, k, pos)
    assert (np.abs(rotated.double().cpu().numpy() - expect_q) <= _bound(q, expect_q, dtype)).all()
    got_k, got_v = _written(cache, slots, ctx, qlens)
    if bits:
        # a code is at most half a step of its group from the row that was quantised; the row itself is off by one rounding
        # of the input type, which can also move the group's bounds: one step covers both, plus the scale's fp16 rounding
        for got, row in ((got_k, expect_k), (got_v, v.double().numpy())):
            grouped = row.reshape(t, hkv, d // 64, 64)
            width = (grouped.max(-1, keepdims=True) - grouped.min(-1, keepdims=True))
            step = np.broadcast_to(width / (2 ** bits - 1), grouped.shape).reshape(row.shape)
            wide = np.broadcast_to(width, grouped.shape).reshape(row.shape)
            assert (np.abs(got - row) <= 0.5 * step + wide * 2.0 ** -10 + np.abs(row).max() * 2 * HALF_STEP[dtype] + 1e-6).all()
        codes, scale, bias = kv_quant.quantize_rows(v.float().numpy(), bits)
        deq = codes.astype(np.float64).reshape(t, hkv, d // 64, 64) * scale[..., None].astype(np.float64) + bias[..., None].astype(np.float64)
        assert np.allclose(got_v, deq.reshape(t, hkv, d), atol=1e-6)
    else:
        assert (np.abs(got_k - expect_k) <= _bound(k, expect_k, dtype)).all()
        assert np.array_equal(got_v, v.double().numpy())
    # nothing else moved
    after = cache.kv_lens.cpu()
    assert [int(after[x]) for x in slots] == [c + n for c, n in zip(ctx, qlens)]
    assert resolved.kv_lens.tolist() == [c + n for c, n in zip(ctx, qlens)]
    assert resolved.query_start_loc.tolist() == [0, *np.cumsum(qlens)]
    assert torch.equal(resolved.block_tables, cache.block_tables[slots])
    touched = torch.zeros(cache.num_blocks, page, dtype=torch.bool)
    bt = cache.block_tables.cpu()
    for i, x in enumerate(slots):
        for p in range(ctx[i], ctx[i] + qlens[i]):
            touched[bt[x, p // page], p % page] = True
    if not bits:
        assert torch.equal(cache.key_cache[~touched], before[0][~touched]) and torch.equal(cache.value_cache[~touched], before[1][~touched])


def test_step_without_advancing_and_a_sequence_that_overflows():
    import easymlx_b200 as emlx

    cache = _cache([10, 250], [4, 4], 2, 64, 16, FP16, 0, [0, 1])
    cache.kv_lens[1] = cache.max_seq_len - 2
    x = torch.ones(8, 2, 64, dtype=FP16, device="cuda")
    meta = emlx.PageMetadata(query_start_loc=emlx.build_query_start_loc([4, 4]), slot_ids=(0, 1),
                             rope_positions=torch.zeros(8, dtype=torch.int32, device="cuda"))
    lens, pool = cache.kv_lens.clone(), cache.key_cache.clone()
    with pytest.raises(RuntimeError, match="outgrows"):
        cache.concatenate_to_cache(x, x, x, cache_metadata=meta, rope=_rope(64), query_lens=[4, 4], advance=False)
    assert torch.equal(cache.kv_lens, lens)
    rows = torch.nonzero((cache.key_cache != pool).flatten(2).any(-1))
    assert rows.shape[0] == 4  # the first sequence's rows only


def test_more_sequences_than_one_launch_serves():
    """Above 2048 sequences the metadata and the rows are two launches; the attention call builds its work list itself."""
    import easymlx_b200 as emlx

    s = 2100
    rng = np.random.default_rng(3)
    ctx = [int(x) for x in rng.integers(0, 40, s)]
    cache = _cache(ctx, [2], 1, 64, 16, FP16, 0, list(range(s)))
    rope = _rope(64)
    q, k, v = (torch.from_numpy(rng.standard_normal((2 * s, h, 64)).astype(np.float32)).to(FP16) for h in (2, 1, 1))
    mask = torch.tensor([[1], [2]] * s, dtype=torch.int64, device="cuda")  # two tokens that both follow the context
    meta = emlx.PageMetadata(query_start_loc=emlx.build_query_start_loc([2] * s), slot_ids=tuple(range(s)), tree_mask=mask)
    rotated, kc, vc, resolved = cache.concatenate_to_cache(q.cuda(), k.cuda(), v.cuda(), cache_metadata=meta, rope=rope, query_lens=[2] * s)
    pos = np.repeat(np.array(ctx, np.int32), 2)[None]
    expect = _expected(rope, q, pos)
    assert (np.abs(rotated.double().cpu().numpy() - expect) <= _bound(q, expect, FP16)).all()
    got_k, got_v = _written(cache, list(range(s)), ctx, [2] * s)
    expect = _expected(rope, k, pos)
    assert (np.abs(got_k - expect) <= _bound(k, expect, FP16)).all() and np.array_equal(got_v, v.double().numpy())
    out = emlx.paged_attention(rotated, kc, vc, resolved.block_tables, resolved.kv_lens, resolved.query_start_loc, softmax_scale=0.125,
                               tree_mask=mask)
    generic = emlx.paged_attention(rotated, kc, vc, resolved.block_tables, resolved.kv_lens, resolved.query_start_loc, softmax_scale=0.125,
                                   tree_mask=mask, kernel="generic")
    assert (out.float() - generic.float()).abs().max() < 8e-3
