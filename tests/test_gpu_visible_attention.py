"""Attention with sinks and over draft trees against a plain 64-bit restatement (run with -m gpu on a B200)."""

import numpy as np
import pytest
import torch

from visible_ref import Batch, attention_bound, check_attention, random_tree

pytestmark = pytest.mark.gpu

FP16, BF16, FP32 = torch.float16, torch.bfloat16, torch.float32
# (hq, hkv, d, page, dtype, bits)
GEOMETRIES = [(8, 2, 64, 16, FP16, 0), (8, 1, 128, 128, BF16, 0), (32, 8, 128, 64, FP16, 0), (6, 2, 128, 32, BF16, 0), (4, 4, 64, 128, FP16, 8),
              (16, 2, 128, 128, BF16, 8), (8, 2, 128, 128, FP16, 4), (12, 1, 64, 128, FP16, 4), (4, 2, 96, 8, FP16, 0),
              (2, 1, 256, 48, BF16, 0), (4, 2, 64, 16, FP32, 0), (40, 8, 64, 128, BF16, 0), (64, 1, 128, 128, FP16, 0)]
KERNELS = ["generic", None]


def _ids(v):
    return "-".join(str(x).replace("torch.", "") for x in v) if isinstance(v, tuple) else str(v)


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("geometry", GEOMETRIES, ids=_ids)
def test_sink_decode(geometry, kernel):
    """Single tokens: contexts below, at and far beyond the window; windows that start inside a page and inside a tile."""
    hq, hkv, d, page, dtype, bits = geometry
    b = Batch([0, 1, 99, 100, 101, 300, 777], [1] * 7, hq, hkv, d, page, dtype, bits, seed=1)
    for window, sinks in ((100, 4), (1, 1), (257, 130), (129, 0), (64, 1000)):
        check_attention(b, d ** -0.5, window, sinks, kernel=kernel)


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("geometry", GEOMETRIES, ids=_ids)
def test_sink_ragged(geometry, kernel):
    """A mixed batch: decode rows, a few tokens, a chunk longer than its window, an absent sequence."""
    hq, hkv, d, page, dtype, bits = geometry
    b = Batch([300, 0, 513, 40, 260], [1, 150, 0, 5, 70], hq, hkv, d, page, dtype, bits, seed=2)
    check_attention(b, d ** -0.5, 90, 5, kernel=kernel)
    check_attention(b, d ** -0.5, 200, 129, kernel=kernel, hints=False)


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("geometry", GEOMETRIES, ids=_ids)
def test_tree(geometry, kernel):
    hq, hkv, d, page, dtype, bits = geometry
    rng = np.random.default_rng(5)
    trees = [random_tree(rng, n) for n in (1, 2, 7, 33, 64)]
    b = Batch([200, 0, 127, 250, 61], [len(t) for t in trees], hq, hkv, d, page, dtype, bits, seed=3, trees=trees)
    check_attention(b, d ** -0.5, kernel=kernel)
    check_attention(b, d ** -0.5, 40, 3, kernel=kernel)
    check_attention(b, d ** -0.5, 3, 1, kernel=kernel)


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("geometry", GEOMETRIES[:3] + GEOMETRIES[5:7], ids=_ids)
def test_trees_beside_causal_rows_and_wide_masks(geometry, kernel):
    hq, hkv, d, page, dtype, bits = geometry
    rng = np.random.default_rng(6)
    trees = [random_tree(rng, 130, forest=False), None, random_tree(rng, 9), None]
    b = Batch([140, 33, 64, 500], [130, 200, 9, 1], hq, hkv, d, page, dtype, bits, seed=4, trees=trees)
    check_attention(b, d ** -0.5, kernel=kernel)
    check_attention(b, d ** -0.5, 70, 10, kernel=kernel)


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("bits", [0, 8, 4])
@pytest.mark.parametrize("q", [1, 3, 40])
def test_invisible_slots_may_hold_nan(bits, q, kernel):
    """Slots past a sequence's end and slots of nobody hold NaN (their scales do in a quantised pool); so do, for single
    tokens, the slots between the sinks and the window, whose pages may serve another sequence by then."""
    b = Batch([260, 5, 390], [q] * 3, 8, 2, 128, 128, FP16, bits, seed=7, poison=float("nan"))
    check_attention(b, 128 ** -0.5, 64, 3, kernel=kernel)
    if q > 1:
        trees = [random_tree(np.random.default_rng(i), q) for i in range(3)]
        check_attention(Batch([260, 5, 390], [q] * 3, 8, 2, 128, 128, FP16, bits, seed=7, poison=float("nan"), trees=trees), 128 ** -0.5, kernel=kernel)
    else:
        for s, n in enumerate(b.kv_lens):
            hidden = [k for k in range(n) if k not in set(b.line(s, 0, 64, 3))]
            for k in hidden:
                at = (int(b.table[s, k // 128]), k % 128)
                if bits:
                    for name in ("k_scale", "k_bias", "v_scale", "v_bias"):
                        b.arrays[name][at[0], :, at[1]] = float("nan")
                else:
                    b.arrays["key"][at], b.arrays["value"][at] = float("nan"), float("inf")
        check_attention(b, 128 ** -0.5, 64, 3, kernel=kernel)


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("hq,hkv,d,dtype,n", [(8, 2, 128, FP16, 4), (8, 2, 64, BF16, 3), (6, 2, 128, FP16, 10), (8, 2, 128, BF16, 40), (16, 2, 64, FP16, 30),
                                              (8, 8, 128, FP16, 12), (8, 2, 64, BF16, 100)])
def test_values_that_are_not_finite_stay_with_the_rows_that_see_them(hq, hkv, d, dtype, n, kernel):
    """A draft whose value row overflowed must not reach its siblings (nor a chunk's later token the earlier ones), while the
    rows that see it do not come out finite."""
    rng = np.random.default_rng(n)
    for window, tree in ((0, True), (45, True), (45, False)):
        b = Batch([150, 301, 20], [n] * 3, hq, hkv, d, 128, dtype, 0, seed=n, trees=[random_tree(rng, n) for _ in range(3)] if tree else None)
        out, mass, reach = b.reference(d ** -0.5, window, 3)
        hit = np.zeros(3 * n, bool)
        for s in range(3):
            ctx = b.ctx[s]
            victims = [ctx + n // 2, ctx + n - 1, ctx - 10, 7]  # two drafts, a context key near the window's edge, one behind the sinks
            for j, key in enumerate(victims):
                b.arrays["value"][int(b.table[s, key // 128]), key % 128, j % hkv, (5 * j) % d] = [float("inf"), float("nan"), float("-inf"), float("nan")][j]
            for i in range(n):
                hit[s * n + i] = bool(set(b.line(s, i, window, 3)) & set(victims))
        got = b.call(d ** -0.5, window, 3, kernel=kernel).double().cpu().numpy()
        fine = np.abs(got - out) <= attention_bound(b, out, mass, reach)
        assert fine[~hit].all()
        assert (~np.isfinite(got)).reshape(3 * n, -1).any(-1)[hit].all()


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (12, 1, 64), (32, 1, 128), (64, 1, 64)])
@pytest.mark.parametrize("window", [0, 33])
def test_a_single_draft_that_does_not_see_itself(hq, hkv, d, window, kernel):
    """Trees of one token: a cleared bit hides the token's own row, whatever it holds, and widens the window by one."""
    b = Batch([130, 128, 40, 0], [1] * 4, hq, hkv, d, 128, FP16, 0, seed=d, trees=[[-1]] * 4)
    b.mask[:] = 0
    b.mask[2] = 1
    out, mass, reach = b.reference(d ** -0.5, window, 2)
    for s in (0, 1, 3):
        b.arrays["value"][int(b.table[s, b.ctx[s] // 128]), b.ctx[s] % 128] = float("nan")
    got = b.call(d ** -0.5, window, 2, kernel=kernel).double().cpu().numpy()
    assert (np.abs(got - out) <= attention_bound(b, out, mass, reach)).all()
    assert (got[3] == 0).all()


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("page", [16, 128])
def test_released_pages_between_sinks_and_window(page, kernel):
    """Pages that no row of the sequence sees any more may be gone from the table."""
    b = Batch([900, 700], [1, 1], 8, 2, 64, page, FP16, 0, seed=8)
    out, mass, reach = b.reference(0.125, 130, 3)
    for s, n in enumerate(b.kv_lens):
        seen = {k // page for k in b.line(s, 0, 130, 3)}
        for i in range(b.mb):
            if i not in seen:
                b.table[s, i] = -1
    got = b.call(0.125, 130, 3, kernel=kernel)  # would raise on a bad page
    assert (np.abs(got.double().cpu().numpy() - out) <= attention_bound(b, out, mass, reach)).all()


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("geometry", [GEOMETRIES[0], GEOMETRIES[2], GEOMETRIES[5]], ids=_ids)
def test_rows_that_see_nothing_are_zero(geometry, kernel):
    hq, hkv, d, page, dtype, bits = geometry
    trees = [[-1, 0, 1], random_tree(np.random.default_rng(0), 40)]
    b = Batch([0, 130], [3, 40], hq, hkv, d, page, dtype, bits, seed=9, trees=trees)
    b.mask[0] = 0            # no context and no token: empty
    b.mask[2] = 0b010        # sees its parent only
    b.mask[5] = 0            # sees the context only
    b.mask[6] = -1           # bits past the sequence's tokens do not count
    got = check_attention(b, d ** -0.5, kernel=kernel)
    assert (got[0] == 0).all() and (got[1] != 0).any()


@pytest.mark.parametrize("bits", [0, 8])
def test_long_contexts_are_split_and_joined(bits):
    """Few sequences with long contexts: the keys are dealt over CTAs and the states combined; twice with equal bits."""
    rng = np.random.default_rng(10)
    trees = [random_tree(rng, 17), random_tree(rng, 64)]
    b = Batch([9001, 3333], [17, 64], 8, 2, 128, 128, BF16, bits, seed=11, trees=trees)
    one = check_attention(b, 128 ** -0.5)
    assert torch.equal(one, b.call(128 ** -0.5))
    c = Batch([9001, 3333], [1, 2], 8, 2, 128, 128, FP16, bits, seed=12)
    one = check_attention(c, 128 ** -0.5, 5000, 7)
    assert torch.equal(one, c.call(128 ** -0.5, 5000, 7))


def test_large_scores_and_one_dominant_key():
    trees = [random_tree(np.random.default_rng(3), 20)]
    check_attention(Batch([1500], [20], 8, 2, 128, 128, FP16, 0, seed=13, trees=trees, k_scale=8.0), 128 ** -0.5)
    check_attention(Batch([1500], [1], 8, 2, 128, 128, FP16, 0, seed=13, k_scale=8.0), 128 ** -0.5, 700, 4)


def test_sinks_without_a_window_change_nothing():
    b = Batch([300, 20], [1, 40], 8, 2, 64, 128, FP16, 0, seed=14)
    assert torch.equal(b.call(0.125, 0, 5), b.call(0.125, 0, 0))


def test_views_and_other_integer_types():
    """Queries, masks and tables that are slices of larger tensors."""
    b = Batch([200, 90], [20, 20], 8, 2, 64, 128, FP16, 0, seed=15, trees=[random_tree(np.random.default_rng(i), 20) for i in (1, 2)])
    from easymlx_b200 import paged_attention

    wide = torch.zeros(40, 8, 67, dtype=FP16, device="cuda")
    wide[..., 3:] = b.q.cuda()
    mask = torch.full((40, 3), -1, dtype=torch.int64, device="cuda")
    mask[:, 1:2] = b.mask.cuda()
    args = (torch.from_numpy(b.table).cuda().long(), torch.from_numpy(b.kv_lens).tolist(), torch.from_numpy(b.qsl).cuda().short())
    got = paged_attention(wide[..., 3:], b.arrays["key"].cuda(), b.arrays["value"].cuda(), *args, softmax_scale=0.125,
                          tree_mask=mask[:, 1:2], tree_seqs=[1, 1])
    assert torch.equal(got, b.call(0.125))


def test_a_tree_wider_than_its_mask_is_reported():
    b = Batch([50], [70], 8, 2, 64, 128, FP16, 0, seed=16, trees=[random_tree(np.random.default_rng(1), 70)])
    b.mask = b.mask[:, :1].contiguous()
    with pytest.raises(RuntimeError, match="mask"):
        b.call(0.125, hints=False)
    with pytest.raises(ValueError, match="mask words"):
        b.call(0.125)
    b.kv_lens[0] = 120  # the status word was reported once; the next call is clean
    b.mask = torch.cat([b.mask, torch.zeros_like(b.mask)], 1)
    b.call(0.125)


def test_two_streams_at_once():
    bs = [Batch([700 * (i + 1)], [30], 8, 2, 128, 128, FP16, 0, seed=20 + i, trees=[random_tree(np.random.default_rng(i), 30)]) for i in range(2)]
    expect = [b.call(0.1) for b in bs]
    streams = [torch.cuda.Stream() for _ in bs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(3):
        for i, (b, s) in enumerate(zip(bs, streams)):
            with torch.cuda.stream(s):
                got[i].append(b.call(0.1))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(expect[i], g) for g in got[i])
