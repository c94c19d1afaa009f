"""Plain 64-bit restatements of sink-window attention, draft-tree attention, multi-axis rotation and tree commits, and
error bounds for the kernels that compute them."""

import numpy as np
import torch

from gpu_util import quantized_pool_from_float
from oracle import kv_quant

HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


class Batch:
    """A packed batch over a shuffled page pool, with 64-bit copies of everything the kernels are given.

    ``ctx`` / ``qlens`` per sequence; ``trees`` is a list of parent lists (``None``: causal rows).  Slots that no sequence
    owns hold ``poison``."""

    def __init__(self, ctx, qlens, hq, hkv, d, page, dtype=torch.float16, bits=0, seed=0, trees=None, poison=None, k_scale=1.0,
                 v_mean=0.0):
        from easymlx_b200 import build_tree_mask

        rng = np.random.default_rng(seed)
        self.ctx, self.qlens, self.hq, self.hkv, self.d, self.page = list(ctx), list(qlens), hq, hkv, d, page
        self.dtype, self.bits, self.trees = dtype, bits, trees
        s, t = len(ctx), int(sum(qlens))
        total = [c + q for c, q in zip(ctx, qlens)]
        per = [max(1, -(-n // page)) for n in total]
        self.mb = max(per) + 1
        nb = sum(per) + 2
        ids = rng.permutation(nb)
        self.table = np.full((s, self.mb), -1, np.int32)
        at = 0
        for i, n in enumerate(per):
            self.table[i, :n] = ids[at:at + n]
            at += n

        def values(*shape):
            return torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).to(dtype)

        self.q = values(t, hq, d)
        k, v = values(nb, page, hkv, d) * k_scale, values(nb, page, hkv, d) + v_mean
        owned = np.zeros((nb, page), bool)
        for i, n in enumerate(total):
            pos = np.arange(n)
            owned[self.table[i, pos // page], pos % page] = True
        self.owned = torch.from_numpy(owned)
        if bits:
            arrays = quantized_pool_from_float(k.float().numpy(), v.float().numpy(), bits)
            names = ("key", "value", "k_scale", "k_bias", "v_scale", "v_bias")
            self.arrays = {n: torch.from_numpy(np.ascontiguousarray(a)) for n, a in zip(names, arrays)}
            if poison is not None:  # the codes of a slot cannot be NaN, its scales and biases can
                where = (~self.owned)[:, None, :, None].expand(nb, hkv, page, d // 64)
                for n in names[2:]:
                    self.arrays[n][where] = poison
            kf = kv_quant.dequantize_key_pool(arrays[0], arrays[2], arrays[3], bits).astype(np.float64)
            vf = kv_quant.dequantize_value_pool(arrays[1], arrays[4], arrays[5], bits).astype(np.float64)
            self.k64, self.v64 = kf, vf
            # a quantised row is scale * code + bias, and the kernels sum the two products apart: what is rounded (and summed)
            # is as large as |scale * code| and |bias| are, however small their sum is
            kb, vb = (np.repeat(a.astype(np.float64).transpose(0, 2, 1, 3), 64, -1) for a in (arrays[3], arrays[5]))
            self.kabs, self.vabs = np.abs(kf - kb) + np.abs(kb), np.abs(vf - vb) + np.abs(vb)
        else:
            if poison is not None:
                k[~self.owned] = poison
                v[~self.owned] = poison
            self.arrays = {"key": k, "value": v}
            self.k64, self.v64 = k.double().numpy(), v.double().numpy()
            self.kabs, self.vabs = np.abs(self.k64), np.abs(self.v64)
        self.kv_lens = np.asarray(total, np.int32)
        self.qsl = np.concatenate([[0], np.cumsum(qlens)]).astype(np.int32)
        self.mask = self.tree_seqs = None
        if trees is not None:
            plain = [p if p is not None else [-1] * min(q, 64) for p, q in zip(trees, qlens)]
            words = max(1, max(-(-q // 64) for p, q in zip(trees, qlens) if p is not None))
            rows = [build_tree_mask([p]) for p in plain]
            self.mask = torch.zeros(t, words, dtype=torch.int64)
            for i, r in enumerate(rows):
                if trees[i] is not None:
                    self.mask[self.qsl[i]:self.qsl[i] + r.shape[0], :r.shape[1]] = r
                else:
                    self.mask[self.qsl[i]:self.qsl[i + 1]] = -1  # must not be read
            if any(p is None for p in trees):
                self.tree_seqs = torch.tensor([p is not None for p in trees])

    def rows(self, s):
        """K and V of sequence ``s`` in slot order, 64 bits, ``[kv_len, Hkv, D]``, and the sizes of what they are summed from."""
        pos = np.arange(int(self.kv_lens[s]))
        at = (self.table[s, pos // self.page], pos % self.page)
        return self.k64[at], self.v64[at], self.kabs[at], self.vabs[at]

    def line(self, s, i, window, sinks):
        """Visible keys of row ``i`` of sequence ``s``, in order."""
        ctx = int(self.kv_lens[s]) - self.qlens[s]
        if self.trees is not None and self.trees[s] is not None:
            words = [int(x) & (2 ** 64 - 1) for x in self.mask[self.qsl[s] + i]]
            new = [j for j in range(self.qlens[s]) if j // 64 < len(words) and words[j // 64] >> (j % 64) & 1]
        else:
            new = list(range(i + 1))
        keys = [*range(ctx), *(ctx + j for j in new)]
        n = len(keys)
        return [k for r, k in enumerate(keys) if not window or r >= n - window or r < sinks]

    def reference(self, scale, window=0, sinks=0):
        """``(out, weight of |v|, largest sum of |q||k| times scale per row)``, all ``[T, Hq, ...]``."""
        t = int(self.qsl[-1])
        out, mass = np.zeros((t, self.hq, self.d)), np.zeros((t, self.hq, self.d))
        reach = np.zeros((t, self.hq, 1))
        g = self.hq // self.hkv
        q = self.q.double().numpy()
        for s in range(len(self.ctx)):
            k, v, kabs, vabs = self.rows(s)
            for i in range(self.qlens[s]):
                keys = self.line(s, i, window, sinks)
                if not keys:
                    continue
                row = q[self.qsl[s] + i].reshape(self.hkv, g, self.d)
                sc = np.einsum("hgd,nhd->hgn", row, k[keys]) * scale
                w = np.exp(sc - sc.max(-1, keepdims=True))
                w /= w.sum(-1, keepdims=True)
                out[self.qsl[s] + i] = np.einsum("hgn,nhd->hgd", w, v[keys]).reshape(self.hq, self.d)
                mass[self.qsl[s] + i] = np.einsum("hgn,nhd->hgd", w, vabs[keys]).reshape(self.hq, self.d)
                reach[self.qsl[s] + i, :, 0] = (np.einsum("hgd,nhd->hgn", np.abs(row), kabs[keys]).max(-1) * scale).reshape(-1)
        return out, mass, reach

    def call(self, scale, window=0, sinks=0, kernel=None, hints=True, **kw):
        from easymlx_b200 import paged_attention

        dev = {n: a.cuda() for n, a in self.arrays.items()}
        extra = {n: a for n, a in dev.items() if n not in ("key", "value")}
        if hints:
            extra.update(max_query_len=max(self.qlens), query_len_set=tuple(sorted({q for q in self.qlens if q})))
        return paged_attention(self.q.cuda(), dev["key"], dev["value"], torch.from_numpy(self.table).cuda(),
                               torch.from_numpy(self.kv_lens).cuda(), torch.from_numpy(self.qsl).cuda(), softmax_scale=scale,
                               sliding_window=window, sink_tokens=sinks, kernel=kernel,
                               tree_mask=None if self.mask is None else self.mask.cuda(),
                               tree_seqs=None if self.tree_seqs is None else self.tree_seqs.cuda(), **extra, **kw)


def attention_bound(batch, out, mass, reach, expanded=False):
    """Largest error a kernel may have, element by element.

    A weight is rounded once to the 16-bit type of the product with V (half a step u of itself, so u * sum w |v| in the
    sum), the output once more (u |out|).  Over a quantised pool v = scale * code + bias: the product of weight and scale is
    what is rounded, so |v| is replaced by |scale * code| + |bias| there (and |k| likewise in the scores).  A score is a 32-bit sum of D products: off by at most D 2^-24 sum |q||k| scale,
    and a score that is off by e changes every normalised weight by at most a factor 1 + 2e (to first order, numerator and
    denominator).  The exponentials (2^-22) and the 32-bit sums over the keys in blocks (2^-20 allows 16 roundings of the
    running values) come on top.  ``expanded``: rows of a quantised pool that were rounded to fp16 first, which moves a
    score by at most 2^-11 sum |q||k| scale and a value by 2^-11 of itself.  Values of bf16 queries over a quantised pool
    pass through fp16 (2^-11 of the row again on the way out)."""
    u = HALF_STEP[batch.dtype]
    pu = u if not batch.bits else 2.0 ** -11
    score = batch.d * 2.0 ** -24 * reach
    if expanded:
        score = score + 2.0 ** -11 * reach
        pu = 2 * pu
    rounding = pu + 2 * score + 2.0 ** -20
    if batch.dtype == torch.float32:
        rounding = 2 * score + 2.0 ** -18
    extra = 2.0 ** -11 * np.abs(out) if batch.bits and batch.dtype == torch.bfloat16 else 0.0
    return rounding * mass * 1.05 + u * np.abs(out) * 1.05 + extra + 1e-7


def check_attention(batch, scale, window=0, sinks=0, expanded=None, **kw):
    out, mass, reach = batch.reference(scale, window, sinks)
    got = batch.call(scale, window, sinks, **kw)
    assert got.dtype == batch.dtype and got.shape == batch.q.shape
    expanded = bool(batch.bits) if expanded is None else expanded
    err, bound = np.abs(got.double().cpu().numpy() - out), attention_bound(batch, out, mass, reach, expanded)
    worst = np.unravel_index(np.nanargmax(np.where(np.isnan(err), np.inf, err - bound)), err.shape)
    assert not np.isnan(err).any() and (err <= bound).all(), f"at {worst}: off by {err[worst]:.3e}, allowed {bound[worst]:.3e}"
    return got


def random_tree(rng, n, forest=True):
    """Parents of a random tree of ``n`` tokens; with ``forest`` several tokens may follow the context directly."""
    return [-1 if i == 0 else int(rng.integers(-1 if forest else 0, i)) for i in range(n)]


def rotate(x, positions, freqs, axis_of_pair, dims, scale=1.0, traditional=False, mscale=1.0):
    """Rotation in 64 bits of ``x [T, H, D]`` at ``positions [axes, T]``."""
    x = np.asarray(x, np.float64).copy()
    angle = positions[axis_of_pair].T.astype(np.float64) * scale / np.asarray(freqs, np.float64)
    cos, sin = np.cos(angle)[:, None], np.sin(angle)[:, None]
    a = (slice(0, dims, 2), slice(1, dims, 2)) if traditional else (slice(0, dims // 2), slice(dims // 2, dims))
    u, v = x[..., a[0]] * mscale, x[..., a[1]] * mscale
    x[..., a[0]], x[..., a[1]] = u * cos - v * sin, u * sin + v * cos
    return x
