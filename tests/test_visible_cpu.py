"""Sinks, draft trees, given rotary positions and commits: what the host checks and builds, without a GPU."""

import ctypes

import numpy as np
import pytest
import torch

import easymlx_b200 as emlx
from easymlx_b200 import _native
from easymlx_b200.caching.paged.cache import tree_arguments
from easymlx_b200.layers.rotary import MultiAxisRotaryEmbedding, RotaryEmbedding, get_rope


@pytest.fixture(scope="module")
def lib():
    from easymlx_b200 import build

    build.build()
    return _native.lib()


def test_tree_mask_of_parents():
    mask = emlx.build_tree_mask([[-1, 0, 0, 2], [], [-1, -1]])
    assert mask.dtype == torch.int64 and mask[:, 0].tolist() == [1, 3, 5, 13, 1, 2]
    chain = emlx.build_tree_mask([[i - 1 for i in range(130)]])
    assert chain.shape == (130, 3)
    assert chain[63].tolist() == [-1, 0, 0] and chain[64].tolist() == [-1, 1, 0] and chain[129].tolist() == [-1, -1, 3]
    assert emlx.build_tree_mask([]).shape == (0, 1)
    for bad in ([[0]], [[-1, 1]], [[-1, 5]], [[-2]]):
        with pytest.raises(ValueError, match="parent"):
            emlx.build_tree_mask(bad)
    with pytest.raises(ValueError, match="4096"):
        emlx.build_tree_mask([[-1] * 4097])


def test_tree_arguments_are_checked():
    cpu = torch.device("cpu")
    good = torch.zeros(4, 2, dtype=torch.int64)
    mask, seqs = tree_arguments(good, [True, False], 4, 2, cpu)
    assert mask is not None and seqs.dtype == torch.int32 and seqs.tolist() == [1, 0]
    assert tree_arguments(good.expand(4, 2)[:, :1], None, 4, 2, cpu)[0].is_contiguous()
    for bad in (good.int(), good[0], good.float(), [[1]], good[:3], torch.zeros(4, 65, dtype=torch.int64), torch.zeros(4, 0, dtype=torch.int64)):
        with pytest.raises(ValueError, match="tree_mask"):
            tree_arguments(bad, None, 4, 2, cpu)
    for bad in ([1], torch.zeros(2), torch.zeros(2, 1, dtype=torch.int32)):
        with pytest.raises(ValueError, match="tree_seqs"):
            tree_arguments(good, bad, 4, 2, cpu)
    with pytest.raises(ValueError, match="needs a tree_mask"):
        tree_arguments(None, [1, 0], 4, 2, cpu)


def test_metadata_carries_the_new_fields():
    mask = torch.ones(1, 1, dtype=torch.int64)
    meta = emlx.PageMetadata(query_start_loc=[0, 1], sink_tokens=3, tree_mask=mask, tree_seqs=[1], rope_positions=[5])
    for other in (meta.with_sliding_window(7), meta.with_cache_state(block_tables=None, kv_lens=None, block_size=16)):
        assert other.sink_tokens == 3 and other.tree_mask is mask and other.tree_seqs == [1] and other.rope_positions == [5]
    assert emlx.PageMetadata(query_start_loc=None) == emlx.PageMetadata(query_start_loc=None, sink_tokens=3)


def test_axes_of_pairs():
    block = MultiAxisRotaryEmbedding(16, sections=(2, 3, 3))
    assert block._axis_of_pair.tolist() == [0, 0, 1, 1, 1, 2, 2, 2]
    turn = MultiAxisRotaryEmbedding(20, sections=(4, 3, 3), interleaved=True)
    assert turn._axis_of_pair.tolist() == [0, 1, 2, 0, 1, 2, 0, 1, 2, 0]
    for bad in ((2, 3), (9, -1), ()):
        with pytest.raises(ValueError, match="sections"):
            MultiAxisRotaryEmbedding(16, sections=bad)
    with pytest.raises(ValueError, match="interleaved"):
        MultiAxisRotaryEmbedding(16, sections=(0, 8), interleaved=True)
    rope = get_rope(128, 1e6, False, {"type": "mrope", "mrope_section": [16, 24, 24]})
    assert isinstance(rope, MultiAxisRotaryEmbedding) and rope.sections == (16, 24, 24) and not rope.interleaved
    assert np.array_equal(rope.freqs, RotaryEmbedding(128, base=1e6).freqs)
    assert get_rope(128, 1e6, False, {"type": "mrope", "mrope_section": [24, 20, 20], "mrope_interleaved": True}).interleaved
    assert type(get_rope(128, 1e6, False, {"type": "mrope"})) is RotaryEmbedding


def test_positions_are_checked():
    rope, cpu = MultiAxisRotaryEmbedding(16, sections=(2, 3, 3)), torch.device("cpu")
    assert rope.checked_positions(torch.arange(4), 4, cpu).shape == (1, 4)
    assert rope.checked_positions([[1, 2]] * 3, 2, cpu).dtype == torch.int32
    for bad in (torch.arange(5), torch.zeros(2, 4, dtype=torch.int64), torch.zeros(4), torch.zeros(3, 4, 1, dtype=torch.int32),
                torch.zeros(4, dtype=torch.bool)):
        with pytest.raises(ValueError, match="positions"):
            rope.checked_positions(bad, 4, cpu)
    with pytest.raises(ValueError, match="positions"):
        RotaryEmbedding(16).checked_positions(torch.zeros(3, 4, dtype=torch.int64), 4, cpu)
    assert rope.inv_freq64(cpu).dtype == torch.float64


def test_struct_layouts_match_the_header():
    assert ctypes.sizeof(_native.Visibility) == 24
    assert ctypes.sizeof(_native.Axes) == 40 and _native.Axes.axis_stride.offset == 24
    assert ctypes.sizeof(_native.StepArgs) == 15 * 8 + 10 * 4 and _native.StepArgs.in_dtype.offset == 120
    assert ctypes.sizeof(_native.CommitLayer) == 9 * 8 + 8


def _pool(**kw):
    p = _native.Pool()
    p.key_cache = p.value_cache = 4096
    p.num_blocks, p.block_size, p.num_kv_heads, p.head_dim = 4, 128, 2, 128
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def test_calls_are_refused_on_the_host(lib):
    """Every refusal comes before any CUDA call, with the pointers never followed."""
    inv, uns, work = _native.EMLX_ERR_INVALID, _native.EMLX_ERR_UNSUPPORTED, _native.EMLX_ERR_WORKSPACE
    vis = _native.Visibility()
    args = _native.AttnArgs()
    args.num_q_heads, args.q_dtype = 4, _native.F16
    assert lib.emlx_attn_visible_generic(args, _pool(), None, None) == inv
    assert lib.emlx_attn_visible_generic(args, _pool(), vis, None) == _native.EMLX_OK  # no tokens
    vis.sink_tokens = -1
    assert lib.emlx_attn_visible_generic(args, _pool(), vis, None) == inv
    vis.sink_tokens, vis.tree_mask, vis.tree_words = 0, 8, 65
    assert lib.emlx_attn_visible_generic(args, _pool(), vis, None) == inv
    vis.tree_words, vis.tree_mask = 1, 12
    assert lib.emlx_attn_visible_generic(args, _pool(), vis, None) == inv
    vis.tree_mask, args.sliding_window = 8, -1
    assert lib.emlx_attn_visible_generic(args, _pool(), vis, None) == inv
    args.sliding_window = 0
    assert lib.emlx_attn_visible_generic(args, _pool(head_dim=512), vis, None) == uns
    n = lib.emlx_visible_plan_bytes(4, 64, 8, 2, 1)
    assert n > lib.emlx_attn_plan_bytes(4, 64, 8, 2) and lib.emlx_visible_plan_bytes(4, 64, 8, 0, 1) == 0
    assert lib.emlx_visible_plan(8, 8, 4, 64, 8, 2, 128, 0, vis, 0, 0, 16, n - 1, None, None) == work
    assert lib.emlx_visible_plan(8, 8, 4, 64, 8, 2, 48, 0, vis, 0, 0, 16, n, None, None) == uns
    assert lib.emlx_visible_plan(8, 8, 4, 64, 7, 2, 128, 0, vis, 0, 0, 16, n, None, None) == inv
    assert lib.emlx_visible_plan(8, 8, 4, 64, 8, 2, 128, 0, vis, 0, 0, 8, n, None, None) == inv  # misaligned

    step = _native.StepArgs()
    assert lib.emlx_positioned_step(step, _pool(), None, None, None, None) == _native.EMLX_OK  # no sequences
    step.num_seqs = 3000
    assert lib.emlx_positioned_step(step, _pool(), None, None, None, None) == uns
    step.num_seqs, step.total_tokens, step.num_slots, step.max_blocks_per_seq = 2, 3, 2, 1
    assert lib.emlx_positioned_step(step, _pool(), None, None, None, None) == inv  # three tokens, no query lengths
    step.total_tokens = 2
    assert lib.emlx_positioned_step(step, _pool(), None, None, None, None) == inv  # NULL arguments
    for name in ("keys", "values", "slot_ids", "block_tables_all", "kv_lens_all", "query_start_loc", "block_tables", "kv_lens", "ticket"):
        setattr(step, name, 4096)
    rope, axes = _native.Rope(), _native.Axes()
    rope.dims = 130
    axes.inv_freq = 4096
    assert lib.emlx_positioned_step(step, _pool(), rope, axes, None, None) == inv
    rope.dims = 128
    assert lib.emlx_positioned_step(step, _pool(), rope, None, None, None) == inv
    axes.positions, axes.num_axes, axes.axis_stride = 4096, 3, 1
    assert lib.emlx_positioned_step(step, _pool(), rope, axes, None, None) == inv
    assert lib.emlx_positioned_write(None, None, 0, None, None, 0, 4, None, None, None, 0, None, None, None, None, None, None) == inv

    layers = (_native.CommitLayer * 1)()
    assert lib.emlx_commit_tree(ctypes.addressof(layers), 1, _pool(), 8, 1, 8, 2, 1, 1, 8, 8, None, None) == inv  # a layer without pointers
    layers[0].key_cache = layers[0].value_cache = layers[0].block_tables = layers[0].kv_lens = 4096
    layers[0].num_blocks = 4
    assert lib.emlx_commit_tree(ctypes.addressof(layers), 0, _pool(), 8, 1, 8, 2, 1, 1, 8, 8, None, None) == inv
    assert lib.emlx_commit_tree(ctypes.addressof(layers), 1, _pool(), None, 1, 8, 2, 1, 1, 8, 8, None, None) == inv
    assert lib.emlx_commit_tree(ctypes.addressof(layers), 1, _pool(), None, 0, None, 0, 1, 1, None, None, None, None) == _native.EMLX_OK


def test_cpu_tensors_are_refused():
    q = torch.zeros((1, 2, 64), dtype=torch.float16)
    kc = torch.zeros((1, 128, 1, 64), dtype=torch.float16)
    with pytest.raises(RuntimeError, match="no CPU path"):
        emlx.paged_attention(q, kc, kc, torch.zeros((1, 1), dtype=torch.int32), torch.ones(1, dtype=torch.int32),
                             torch.tensor([0, 1], dtype=torch.int32), tree_mask=torch.ones(1, 1, dtype=torch.int64))
    with pytest.raises(ValueError, match="sink_tokens"):
        emlx.paged_attention(q, kc, kc, None, None, None, sink_tokens=-1)
