"""Measured cases of the paged step's operators beyond a plain causal sequence.

Four operators, each in a plain form (elementary torch operations) and through the framework's own calls:

* ``sink``    attention with a sliding window over the paged cache in which the first tokens stay visible;
* ``tree``    attention of a tree of drafted tokens over the paged cache (each node sees the context and its ancestors);
* ``rope``    the cache write of a step whose rotary positions are given, one per token and axis (time, height, width);
* ``commit``  keeping a tree's accepted path: its rows move to the end of the context, in every layer's cache.

A row's *visible sequence* is the context followed by the new keys whose mask bit is set (a causal row: those up to
itself).  A sliding window keeps its last ``window`` entries, sinks keep its first ``sinks`` ones.
"""

import math

import numpy as np
import torch

own = False

HALF = {"fp16": torch.float16, "bf16": torch.bfloat16, "affine8": torch.float16, "affine4": torch.float16}


def listed():
    return [
        # one sequence of a chat that outgrew its window, one new token: latency
        dict(name="sink_decode_one", op="sink", seqs=1, q=1, ctx_lo=8191, ctx_hi=8191, hq=32, hkv=8, d=128, kind="fp16",
             page=16, window=1024, sinks=4, step=True),
        # a full decode batch with the cache in 8-bit codes, a window larger than some of the contexts
        dict(name="sink_decode_batch", op="sink", seqs=160, q=1, ctx_lo=1023, ctx_hi=8191, hq=64, hkv=8, d=128,
             kind="affine8", page=128, window=4096, sinks=64, step=False),
        # prefill chunks of two long prompts, bf16, ragged lengths, pages smaller than a tile
        dict(name="sink_prefill", op="sink", seqs=2, q=2041, ctx_lo=5003, ctx_hi=14011, hq=32, hkv=8, d=128, kind="bf16",
             page=64, window=4096, sinks=16, step=False),
        # one user, a small tree after a short context: latency
        dict(name="tree_one", op="tree", seqs=1, q=16, ctx_lo=2045, ctx_hi=2045, hq=32, hkv=8, d=128, kind="fp16", page=128,
             window=0, sinks=0, step=True),
        # one user with a long document, the widest tree of one mask word
        dict(name="tree_long", op="tree", seqs=1, q=64, ctx_lo=32749, ctx_hi=32749, hq=64, hkv=8, d=128, kind="bf16",
             page=128, window=0, sinks=0, step=True),
        # a serving batch verifying one tree per sequence
        dict(name="tree_batch", op="tree", seqs=48, q=27, ctx_lo=512, ctx_hi=8192, hq=32, hkv=8, d=128, kind="fp16",
             page=128, window=0, sinks=0, step=True),
        # head size 64, window and sinks under a tree
        dict(name="tree_window", op="tree", seqs=24, q=40, ctx_lo=700, ctx_hi=9001, hq=32, hkv=8, d=64, kind="fp16", page=32,
             window=2048, sinks=8, step=True),
        # the cache in 8-bit codes
        dict(name="tree_affine8", op="tree", seqs=16, q=24, ctx_lo=1030, ctx_hi=8191, hq=32, hkv=8, d=128, kind="affine8",
             page=128, window=0, sinks=0, step=False),
        # decode step of a vision-language model: one token per sequence, three position axes
        dict(name="rope_decode", op="rope", seqs=64, q=1, ctx_lo=200, ctx_hi=4000, hq=32, hkv=8, d=128, kind="bf16", page=128,
             sections="16,24,24", interleaved=False),
        # prefill of prompts with images, interleaved axes
        dict(name="rope_prefill", op="rope", seqs=4, q=2047, ctx_lo=0, ctx_hi=3000, hq=64, hkv=8, d=128, kind="bf16", page=16,
             sections="24,20,20", interleaved=True),
        # one user: the accepted path in every layer of a small model
        dict(name="commit_one", op="commit", layers=16, seqs=1, q=16, most=5, ctx_lo=411, ctx_hi=411, hkv=8, d=64, kind="fp16",
             page=16),
        # a serving batch
        dict(name="commit_batch", op="commit", layers=24, seqs=64, q=32, most=8, ctx_lo=64, ctx_hi=700, hkv=8, d=128,
             kind="bf16", page=128),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["sink", "sink", "tree", "tree", "rope", "commit"])
    hq, hkv = rng.choice([(32, 8), (64, 8), (8, 8), (16, 2), (24, 8), (40, 8), (12, 1)])
    d, page = rng.choice([64, 128]), rng.choice([16, 32, 64, 128])
    if op == "commit":
        q = rng.randint(4, 64)
        return dict(op=op, layers=_log(rng, 2, 24), seqs=_log(rng, 1, 64), q=q, most=rng.randint(1, max(1, min(q // 2, 10))),
                    ctx_lo=_log(rng, 1, 60), ctx_hi=_log(rng, 64, 700), hkv=hkv, d=d, kind=rng.choice(["fp16", "bf16"]), page=page)
    if op == "rope":
        q = _log(rng, 1, 2000)
        a = rng.randint(2, d // 4)
        b = rng.randint(1, d // 2 - a - 1)
        inter = rng.random() < 0.5
        sections = (d // 2 - 2 * (d // 6), d // 6, d // 6) if inter else (a, b, d // 2 - a - b)
        return dict(op=op, seqs=max(1, min(128, _log(rng, 1, 8000) // q)), q=q, ctx_lo=0, ctx_hi=_log(rng, 10, 4000), hq=hq,
                    hkv=hkv, d=d, kind=rng.choice(["fp16", "bf16"]), page=page, sections=",".join(map(str, sections)),
                    interleaved=inter)
    kind = rng.choice(["fp16", "fp16", "bf16", "bf16", "affine8", "affine4"])
    if kind.startswith("affine"):
        page = 128
    if op == "sink":
        q = rng.choice([1, 1, 1, _log(rng, 2, 16), _log(rng, 17, 1500)])
        seqs = max(1, min(128, _log(rng, 1, 128) // max(1, q // 8)))
        hi = _log(rng, 600, 12000)
        return dict(op=op, seqs=seqs, q=q, ctx_lo=rng.randint(0, 500), ctx_hi=hi, hq=hq, hkv=hkv, d=d, kind=kind, page=page,
                    window=_log(rng, 64, 6000), sinks=rng.choice([1, 4, 5, 16, 64, 130]), step=not kind.startswith("affine"))
    q = _log(rng, 2, 64)
    seqs = max(1, min(48, _log(rng, 1, 48)))
    hi = _log(rng, 300, 28000 if seqs <= 2 else 8000)
    windowed = rng.random() < 0.3
    return dict(op=op, seqs=seqs, q=q, ctx_lo=rng.randint(0, 250), ctx_hi=hi, hq=hq, hkv=hkv, d=d, kind=kind, page=page,
                window=_log(rng, 70, 5000) if windowed else 0, sinks=rng.choice([0, 4, 20]) if windowed else 0,
                step=not kind.startswith("affine"))


def _contexts(case):
    """Context length of every sequence: spread over the range, the same for every seed."""
    lo, hi = min(case["ctx_lo"], case["ctx_hi"]), max(case["ctx_lo"], case["ctx_hi"])
    s = np.arange(1, case["seqs"] + 1)
    return (lo + np.floor((hi - lo + 0.999) * ((s * 0.6180339887498949) % 1.0))).astype(np.int64)


def _row_bytes(case):
    bits = {"affine8": 8, "affine4": 4}.get(case["kind"], 16)
    return case["d"] * bits // 8 + (4 * (case["d"] // 64) if bits < 16 else 0)


def work(case):
    ctx, q, hkv, d = _contexts(case), case["q"], case["hkv"], case["d"]
    if case["op"] == "commit":
        moved = case["layers"] * case["seqs"] * hkv * 2 * max(1, case["most"] // 2)
        return {"bytes": 2 * moved * _row_bytes(case), "flops": 0}
    tokens = case["seqs"] * q
    if case["op"] == "rope":
        return {"bytes": tokens * 2 * d * (2 * case["hq"] + 4 * hkv) + 12 * tokens, "flops": 3 * tokens * d * (case["hq"] + hkv)}
    total = ctx + q
    window, sinks = case["window"], case["sinks"]
    if window:
        keys = np.minimum(total, window + q - 1 + sinks)
        rows = np.minimum(ctx + (q + 1) / 2 if case["op"] == "sink" else ctx + 1.0, window + sinks)
    else:
        keys, rows = total, ctx + 1.0
    written = 4 * tokens * hkv * 2 * d if case["step"] else 0
    return {"bytes": int(keys.sum()) * 2 * hkv * _row_bytes(case) + 4 * tokens * case["hq"] * d + written,
            "flops": 4 * case["hq"] * d * q * float(rows.sum())}


# ------------------------------------------------------------------------------------------------------------- inputs
def _tables(rng, totals, page, spare):
    """Page table of the sequences over a shuffled pool with some pages that belong to nobody."""
    per = [-(-int(n) // page) for n in totals]
    pages = sum(per) + spare
    ids = rng.permutation(pages)
    table = np.full((len(totals), max(per)), -1, np.int32)
    at = 0
    for s, n in enumerate(per):
        table[s, :n] = ids[at:at + n]
        at += n
    return table, pages


def _trees(rng, seqs, nodes):
    """Ancestor masks (bit j of word i: node i sees node j) of random trees: parents before children, node 0 the root."""
    mask = np.zeros((seqs, nodes), np.uint64)
    mask[:, 0] = 1
    for i in range(1, nodes):
        parent = np.maximum(0, i - 1 - np.floor(rng.exponential(3.0, seqs)).astype(np.int64))
        mask[:, i] = mask[np.arange(seqs), parent] | (np.uint64(1) << np.uint64(i))
    return mask.view(np.int64)


def _affine_pool(x, bits):
    """Group-64 min-max codes of rows [NB, bs, Hkv, D], in the cache's layout: key codes token-major, value codes with the
    tokens of one element contiguous, scales and biases head-major inside a page."""
    def codes(y):
        nb, bs, h, d = y.shape
        g = y.float().reshape(nb, bs, h, d // 64, 64)
        lo, hi = g.amin(-1), g.amax(-1)
        scale, bias = ((hi - lo) / (2 ** bits - 1)).half(), lo.half()
        scale = torch.where(scale == 0, torch.ones_like(scale), scale)
        c = torch.round((g - bias.float()[..., None]) / scale.float()[..., None]).clamp(0, 2 ** bits - 1)
        return c.reshape(nb, bs, h, d).to(torch.uint8), scale.permute(0, 2, 1, 3).contiguous(), bias.permute(0, 2, 1, 3).contiguous()

    def pack(c):
        return c.contiguous() if bits == 8 else (c[..., 0::2] | (c[..., 1::2] << 4)).contiguous()

    kc, ks, kb = codes(x[0])
    vc, vs, vb = codes(x[1])
    return dict(k=pack(kc), v=pack(vc.permute(0, 2, 3, 1)), k_scale=ks, k_bias=kb, v_scale=vs, v_bias=vb)


def prepare(case, seed):
    dev = torch.device("cuda")
    rng = np.random.RandomState(seed % (2 ** 31))
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype = HALF[case["kind"]]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=dev, dtype=torch.float32).to(dtype)

    ctx, q, hkv, d, page = _contexts(case), case["q"], case["hkv"], case["d"], case["page"]
    seqs, tokens = case["seqs"], case["seqs"] * q
    table, pages = _tables(rng, ctx + q, page, 1 + seqs // 8)
    st = dict(case=case, ctx=torch.tensor(ctx, dtype=torch.int32, device=dev), table=torch.from_numpy(table).to(dev),
              scale=d ** -0.5)
    if case["op"] == "commit":
        most = case["most"]
        accepted = np.full((seqs, most), -1, np.int32)
        accepted[:, 0] = 0
        for s in range(seqs):
            n = rng.randint(1, min(most, q - most + 1) + 1)
            accepted[s, 1:n] = np.sort(rng.choice(np.arange(most, q), n - 1, replace=False))
        st.update(accepted=torch.from_numpy(accepted).to(dev), lens=st["ctx"].clone(),
                  k=[normal(pages, page, hkv, d) for _ in range(case["layers"])],
                  v=[normal(pages, page, hkv, d) for _ in range(case["layers"])])
    else:
        st.update(q=normal(tokens, case["hq"], d), lens=st["ctx"] + q)
        if case["kind"].startswith("affine"):
            st.update(_affine_pool((normal(pages, page, hkv, d), normal(pages, page, hkv, d)), int(case["kind"][6:])))
        else:
            st.update(k=normal(pages, page, hkv, d), v=normal(pages, page, hkv, d), new_k=normal(tokens, hkv, d),
                      new_v=normal(tokens, hkv, d))
        if case["op"] == "tree":
            st["mask"] = torch.from_numpy(_trees(rng, seqs, q).reshape(tokens, 1)).to(dev)
        if case["op"] == "rope":
            # text before and after a picture: on the text the axes agree, on the picture they differ
            base = ctx[:, None] + np.arange(q)[None]
            wide = 1 + rng.randint(0, 64)
            pos = np.stack([base, base + np.arange(q)[None] // wide, base + np.arange(q)[None] % wide])
            st["positions"] = torch.from_numpy(pos.reshape(3, tokens).astype(np.int32)).to(dev)
            st["periods"] = (np.float32(1e6) ** (np.arange(0, d, 2, dtype=np.float32) / np.float32(d))).astype(np.float32)
    if own:
        st["call"] = _own_call(st)
    return st


# ------------------------------------------------------------------------------------------- through the framework
def _own_call(st):
    """What a user's program sets up once: the cache over its buffers, and for a step the captured graph."""
    import easymlx_b200 as emlx
    from easymlx_b200.layers.rotary import MultiAxisRotaryEmbedding
    from easymlx_b200.runtime import AttentionStep

    case = st["case"]
    op, page, hkv, d, seqs, q = case["op"], case["page"], case["hkv"], case["d"], case["seqs"], case["q"]

    def view(k, v, lens, **more):
        return emlx.PageCacheView(key_cache=k, value_cache=v, block_tables=st["table"], kv_lens=lens, block_size=page,
                                  num_kv_heads=hkv, head_dim=d, **more)

    slots = tuple(range(seqs))
    if op == "commit":
        cache = emlx.PageCache([view(k, v, st["lens"]) for k, v in zip(st["k"], st["v"])])
        slot_ids = torch.arange(seqs, dtype=torch.int32, device="cuda")

        def commit():
            lens = cache.commit_tree(slot_ids, st["accepted"], advance=False)
            return {"lens": lens, "k": st["k"], "v": st["v"]}
        return commit
    if op == "rope":
        cache = view(st["k"], st["v"], st["ctx"].clone())
        rope = MultiAxisRotaryEmbedding(d, freqs=st["periods"], sections=tuple(int(x) for x in case["sections"].split(",")),
                                        interleaved=case["interleaved"])
        meta = emlx.PageMetadata(query_start_loc=emlx.build_query_start_loc([q] * seqs), slot_ids=slots,
                                 rope_positions=st["positions"])

        def write():
            return cache.concatenate_to_cache(st["q"], st["new_k"], st["new_v"], cache_metadata=meta, rope=rope,
                                              query_lens=[q] * seqs, advance=False)[0]
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            write()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            rotated = write()

        st["keep"] = (cache, rope, meta)  # the graph reads their tables and lengths

        def replay():
            graph.replay()
            return {"q": rotated, "k": st["k"], "v": st["v"]}
        return replay
    if case["step"]:
        step = AttentionStep(view(st["k"], st["v"], st["ctx"].clone()), st["q"], st["new_k"], st["new_v"], [q] * seqs, slots,
                             scale=st["scale"], sliding_window=case["window"], sink_tokens=case["sinks"],
                             tree_mask=st.get("mask")).capture(warmup=1)
        return lambda: {"out": step.step(), "k": st["k"], "v": st["v"]}
    starts = torch.arange(seqs + 1, dtype=torch.int32, device="cuda") * q
    extra = {x: st[x] for x in ("k_scale", "k_bias", "v_scale", "v_bias") if x in st}
    long_seqs = seqs if q * (case["hq"] // hkv) >= 64 else 0

    def attend():
        return {"out": emlx.paged_attention(
            st["q"], st["k"], st["v"], st["table"], st["lens"], starts, softmax_scale=st["scale"],
            sliding_window=case["window"], sink_tokens=case["sinks"], tree_mask=st.get("mask"), max_query_len=q,
            query_len_set=(q,), long_seqs=long_seqs, **extra)}
    return attend


# ------------------------------------------------------------------------------------------------------- plain form
def _slots(st, positions):
    """Flat pool row of every position [S, n] of the sequences."""
    page = st["case"]["page"]
    idx = (positions // page).clamp(max=st["table"].shape[1] - 1)
    return torch.gather(st["table"].long(), 1, idx).clamp(min=0) * page + positions % page


def _visible(st, length):
    """[S, q, length]: whether row i sees key c."""
    case = st["case"]
    seqs, q, window, sinks = case["seqs"], case["q"], case["window"], case["sinks"]
    ctx = st["ctx"].long()[:, None, None]
    key = torch.arange(length, device="cuda")[None, None]
    row = torch.arange(q, device="cuda")[None, :, None]
    if case["op"] == "tree":
        bit = (st["mask"].view(seqs, q, 1) >> torch.arange(q, device="cuda")[None, None]) & 1
    else:
        bit = (torch.arange(q, device="cuda")[None, None] <= row).long().expand(seqs, q, q)
    count = bit.sum(-1, keepdim=True)
    node = (key - ctx).clamp(0, q - 1)
    rank = torch.where(key < ctx, key.expand(seqs, q, length),
                       ctx + torch.gather(torch.cumsum(bit, -1) - bit, 2, node.expand(seqs, q, length)))
    seen = (key < ctx) | ((key < ctx + q) & (torch.gather(bit, 2, node.expand(seqs, q, length)) == 1))
    if window:
        seen = seen & ((rank >= ctx + count - window) | (rank < sinks))
    return seen


def _rows(st, slots):
    """Keys and values [S, n, Hkv, D] of flat pool rows in 32 bits."""
    case = st["case"]
    if not case["kind"].startswith("affine"):
        return tuple(st[x].reshape(-1, case["hkv"], case["d"])[slots].float() for x in "kv")
    bits, page = int(case["kind"][6:]), case["page"]
    pg, off = slots // page, slots % page

    def unpack(c):
        return c if bits == 8 else torch.stack([c & 15, c >> 4], -1).flatten(-2)

    k = unpack(st["k"])[pg, off].float()
    v = unpack(st["v"]).permute(0, 3, 1, 2)[pg, off].float()

    def per_group(x):
        return x.permute(0, 2, 1, 3)[pg, off].float().repeat_interleave(64, -1)

    return k * per_group(st["k_scale"]) + per_group(st["k_bias"]), v * per_group(st["v_scale"]) + per_group(st["v_bias"])


def _plain_attention(st):
    case = st["case"]
    seqs, q, hq, hkv, d = case["seqs"], case["q"], case["hq"], case["hkv"], case["d"]
    if case["step"]:
        new = _slots(st, st["ctx"].long()[:, None] + torch.arange(q, device="cuda")[None])
        st["k"].view(-1, hkv, d)[new.reshape(-1)] = st["new_k"]
        st["v"].view(-1, hkv, d)[new.reshape(-1)] = st["new_v"]
    length = int(_contexts(case).max()) + q
    k, v = _rows(st, _slots(st, torch.arange(length, device="cuda")[None].expand(seqs, length)))
    queries = st["q"].float().view(seqs, q, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(seqs, hkv, -1, d) * st["scale"]
    scores = queries @ k.permute(0, 2, 3, 1)
    seen = _visible(st, length)[:, None, None]
    scores = torch.where(seen, scores.view(seqs, hkv, hq // hkv, q, length), float("-inf"))
    top = scores.amax(-1, keepdim=True)
    weight = torch.exp(scores - torch.where(top == float("-inf"), torch.zeros_like(top), top))
    total = weight.sum(-1, keepdim=True)
    out = (weight.view(seqs, hkv, -1, length) @ v.permute(0, 2, 1, 3)).view(seqs, hkv, hq // hkv, q, d)
    out = torch.where(total > 0, out / total, torch.zeros_like(out))
    out = out.permute(0, 3, 1, 2, 4).reshape(seqs * q, hq, d).to(st["q"].dtype)
    return {"out": out, "k": st["k"], "v": st["v"]} if case["step"] else {"out": out}


def _axis_of_pair(case):
    sections = [int(x) for x in case["sections"].split(",")]
    pair = np.arange(case["d"] // 2)
    if not case["interleaved"]:
        return np.repeat(np.arange(3), sections)
    return np.where((pair % 3 > 0) & (pair < 3 * np.asarray(sections)[pair % 3]), pair % 3, 0)


def _plain_rope(st):
    case = st["case"]
    half, hkv, d, q = case["d"] // 2, case["hkv"], case["d"], case["q"]
    axis = torch.from_numpy(_axis_of_pair(case)).to("cuda")
    angle = st["positions"].double()[axis].T / torch.from_numpy(st["periods"]).to("cuda").double()
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]

    def rotate(x):
        a, b = x[..., :half].float(), x[..., half:].float()
        return torch.cat([a * cos - b * sin, a * sin + b * cos], -1).to(x.dtype)

    new = _slots(st, st["ctx"].long()[:, None] + torch.arange(q, device="cuda")[None]).reshape(-1)
    st["k"].view(-1, hkv, d)[new] = rotate(st["new_k"])
    st["v"].view(-1, hkv, d)[new] = st["new_v"]
    return {"q": rotate(st["q"]), "k": st["k"], "v": st["v"]}


def _plain_commit(st):
    case = st["case"]
    accepted = st["accepted"].long()
    ctx = st["ctx"].long()[:, None]
    live = accepted >= 0
    source = _slots(st, ctx + accepted.clamp(min=0))[live]
    target = _slots(st, ctx + torch.arange(case["most"], device="cuda")[None])[live]
    pools = [x.view(-1, case["hkv"], case["d"]) for x in st["k"] + st["v"]]
    moved = [x[source] for x in pools]
    [x.index_copy_(0, target, y) for x, y in zip(pools, moved)]
    return {"lens": st["ctx"] + live.sum(-1, dtype=torch.int32), "k": st["k"], "v": st["v"]}


def run(st):
    if own:
        return st["call"]()
    return {"sink": _plain_attention, "tree": _plain_attention, "rope": _plain_rope, "commit": _plain_commit}[st["case"]["op"]](st)


# -------------------------------------------------------------------------------------------- the definition, 64 bits
def _exact_attention(st):
    case = st["case"]
    q, hq, hkv, d, page, group = case["q"], case["hq"], case["hkv"], case["d"], case["page"], case["hq"] // case["hkv"]
    window, sinks = case["window"], case["sinks"]
    out = torch.zeros(case["seqs"] * q, hq, d, dtype=torch.float64, device="cuda")
    for s, ctx in enumerate(_contexts(case).tolist()):
        where = [int(p) for p in st["table"][s].tolist()]
        ids = torch.tensor(where[:-(-(ctx + q) // page)], device="cuda")
        if case["kind"].startswith("affine"):
            bits = int(case["kind"][6:])

            def values(codes, scale, bias, by_token):
                c = codes[ids].to(torch.int64)
                if bits == 4:
                    both = torch.empty(*c.shape[:-1], 2 * c.shape[-1], dtype=torch.int64, device="cuda")
                    both[..., 0::2], both[..., 1::2] = c % 16, c // 16
                    c = both
                c = c if by_token else c.permute(0, 3, 1, 2)
                sc, bi = (y[ids].permute(0, 2, 1, 3).double() for y in (scale, bias))
                grouped = c.double().reshape(len(ids), page, hkv, d // 64, 64)
                return (grouped * sc[..., None] + bi[..., None]).reshape(-1, hkv, d)[:ctx + q]
            k = values(st["k"], st["k_scale"], st["k_bias"], True)
            v = values(st["v"], st["v_scale"], st["v_bias"], False)
        else:
            k, v = (st[x][ids].double().reshape(-1, hkv, d)[:ctx + q] for x in "kv")
            if case["step"]:
                k[ctx:], v[ctx:] = st["new_k"][s * q:(s + 1) * q].double(), st["new_v"][s * q:(s + 1) * q].double()
        for i in range(q):
            line = torch.arange(ctx + i + 1, device="cuda")
            if case["op"] == "tree":
                word = int(st["mask"][s * q + i, 0]) & (2 ** 64 - 1)
                nodes = [ctx + j for j in range(q) if word >> j & 1]
                line = torch.cat([torch.arange(ctx, device="cuda"), torch.tensor(nodes, dtype=torch.int64, device="cuda")])
            first = len(line) - window
            if window and first > 0:
                line = torch.cat([line[:min(sinks, first)], line[first:]])
            rows = st["q"][s * q + i].double().view(hkv, group, d)
            scores = torch.einsum("hgd,nhd->hgn", rows, k[line]) * st["scale"]
            out[s * q + i] = torch.einsum("hgn,nhd->hgd", torch.softmax(scores, -1), v[line]).reshape(hq, d)
    return out


def exact(case, seed):
    op, tokens = case["op"], case["seqs"] * case["q"]
    if op in ("sink", "tree") and tokens > 6000:
        return None
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    if op in ("sink", "tree"):
        out = _exact_attention(st)
        return {"out": out, "k": None, "v": None} if case["step"] else {"out": out}
    if op == "commit":
        lens, table = st["ctx"].long(), st["table"].tolist()
        for pool in st["k"] + st["v"]:
            flat = pool.view(-1, case["hkv"], case["d"])
            for s, (ctx, path) in enumerate(zip(_contexts(case).tolist(), st["accepted"].tolist())):
                path = [a for a in path if a >= 0]
                to, at = ([int(table[s][p // case["page"]]) * case["page"] + p % case["page"] for p in places]
                          for places in ([ctx + j for j in range(len(path))], [ctx + a for a in path]))
                flat[to] = flat[at]
                lens[s] = ctx + len(path)
        return {"lens": lens, "k": [x.double() for x in st["k"]], "v": [x.double() for x in st["v"]]}
    half, q, d, hkv = case["d"] // 2, case["q"], case["d"], case["hkv"]
    sections = [int(x) for x in case["sections"].split(",")]
    axes = []
    for i in range(half):
        if case["interleaved"]:
            axes.append(i % 3 if i % 3 and i < 3 * sections[i % 3] else 0)
        else:
            axes.append(0 if i < sections[0] else 1 if i < sections[0] + sections[1] else 2)
    turn = torch.stack([st["positions"][a].double() / float(p) for a, p in zip(axes, st["periods"])], -1)
    phase = torch.polar(torch.ones_like(turn), turn)[:, None]

    def rotate(x):
        y = torch.complex(x[..., :half].double(), x[..., half:].double()) * phase
        return torch.cat([y.real, y.imag], -1)

    k, v = st["k"].double(), st["v"].double()
    turned = rotate(st["new_k"])
    for s, ctx in enumerate(_contexts(case).tolist()):
        pos = torch.arange(ctx, ctx + q, device="cuda")
        pages = st["table"][s].long()[pos // case["page"]]
        k[pages, pos % case["page"]] = turned[s * q:(s + 1) * q]
        v[pages, pos % case["page"]] = st["new_v"][s * q:(s + 1) * q].double()
    return {"q": rotate(st["q"]), "k": k, "v": v}
