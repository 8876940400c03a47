"""Operator cases of the 4-bit KV cache and of sparse (page-selecting) decode attention.

Each case is one call, or the two calls a program makes together, of an operator
over paged K/V pools, in its plain form (elementary torch operations) or through
this package. Sizes are those of the package's own decode configurations, with
odd head sizes, page sizes and ragged lengths beside them.

4-bit pools are uint8 [num_blocks, Hkv, block_size / 16, 9 * D]: per 16 tokens
the E2M1 codes (16 * D / 2 bytes, two per byte, low nibble first), then the E4M3
scales (one per token and 16 channels). K rows hold, for t = 0..3, the codes of
channels 16 j + 4 t .. + 3 for every j; K scales are [token][D / 16]. V rows are
in channel order; V scales are [D / 16][token].
"""
import math

import numpy as np
import torch

own = False

_DEV = "cuda"
_LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
_SCALES = {"k": 0.011, "v": 0.0073}  # pool scales, as a calibration leaves them


# ── cases ────────────────────────────────────────────────────────────────
def listed():
    return [
        # one decode step of 64 sequences: each one's new token is stored, and read back
        dict(name="store step", op="store", tokens=64, heads=8, dim=128, page=16, pad=0, skip=0),
        # a prompt of 8192 tokens
        dict(name="store prompt", op="store", tokens=8192, heads=8, dim=128, page=16, pad=0, skip=0),
        # odd head size, 32-token pages, rows inside a fused QKV row, some tokens skipped
        dict(name="store odd", op="store", tokens=777, heads=5, dim=80, page=32, pad=1600, skip=7),
        # a small model's short contexts: latency counts
        dict(name="q4 small", op="q4", seqs=4, q_heads=12, heads=12, dim=64, page=16, low=37, high=512),
        # Llama-3-8B decode
        dict(name="q4 decode", op="q4", seqs=64, q_heads=32, heads=8, dim=128, page=16, low=1024, high=8192),
        # Llama-3-70B long contexts
        dict(name="q4 long", op="q4", seqs=8, q_heads=64, heads=8, dim=128, page=16, low=32768, high=131072),
        # odd head size and group, 32-token pages, empty and one-token sequences
        dict(name="q4 odd", op="q4", seqs=13, q_heads=20, heads=4, dim=96, page=32, low=0, high=3001),
        # the summaries after a decode step: each sequence's newest page
        dict(name="bounds step", op="bounds", seqs=64, heads=8, dim=128, page=16, low=1024, high=8192, new=1, fp32=False),
        # the summaries of whole prompts
        dict(name="bounds prompt", op="bounds", seqs=8, heads=8, dim=128, page=16, low=2048, high=32768, new=0, fp32=False),
        # 256 of up to 8192 pages per KV head
        dict(name="sparse long", op="sparse", seqs=8, q_heads=64, heads=8, dim=128, page=16, low=32768, high=131072, keep=256, sink=1, recent=4, fp32=False, q4=False),
        # 64 of up to 512 pages, from the 4-bit cache
        dict(name="sparse q4", op="sparse", seqs=64, q_heads=32, heads=8, dim=128, page=16, low=1024, high=8192, keep=64, sink=1, recent=2, fp32=False, q4=True),
        # fp32 pools, short contexts, some shorter than what is kept
        dict(name="sparse fp32", op="sparse", seqs=5, q_heads=12, heads=12, dim=64, page=16, low=0, high=777, keep=9, sink=0, recent=1, fp32=True, q4=False),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["store", "q4", "q4", "bounds", "sparse", "sparse"])
    heads = rng.choice([1, 2, 3, 4, 5, 8])
    dim = rng.choice([64, 128, 128, 256]) if rng.random() < 0.7 else 16 * rng.randint(2, 16)
    page = rng.choice([16, 16, 16, 32, 64])
    if op == "store":
        tokens = min(_log(rng, 1, 8192), 8192 * 1024 // (heads * dim))
        return dict(op=op, tokens=tokens, heads=heads, dim=dim, page=page, pad=rng.choice([0, 0, 64, 1000]), skip=rng.choice([0, 0, 5]))
    seqs, high = _log(rng, 1, 64), _log(rng, 16, 65536)
    high = max(16, min(high, 8 * 131072 * 1024 // (2 * seqs * heads * dim)))
    low = rng.choice([0, high // 4, high])
    if op == "bounds":
        return dict(op=op, seqs=seqs, heads=heads, dim=dim, page=page, low=low, high=min(high, 8 * 32768 // seqs), new=rng.choice([0, 0, 1, 100]), fp32=rng.random() < 0.3)
    q_heads = heads * rng.choice([1, 2, 3, 4, 8, 16])
    if op == "q4":
        return dict(op=op, seqs=seqs, q_heads=q_heads, heads=heads, dim=dim, page=page, low=low, high=high)
    keep = _log(rng, 4, 256)
    q4 = rng.random() < 0.4
    return dict(op=op, seqs=seqs, q_heads=q_heads, heads=heads, dim=dim, page=page, low=low, high=high, keep=keep, sink=rng.choice([0, 1, 2]),
                recent=rng.choice([1, 2]), fp32=not q4 and rng.random() < 0.3, q4=q4)


def _lens(case, seed):
    """Context lengths between low and high; the first sequence has the longest."""
    rng = np.random.default_rng(seed)
    lens = rng.integers(case["low"], case["high"] + 1, size=case["seqs"])
    lens[0] = case["high"]
    if case["low"] == 0 and len(lens) > 2:
        lens[1], lens[2] = 0, 1
    return lens


# ── the 4-bit format ─────────────────────────────────────────────────────
def _const(x):
    return torch.full((), x, dtype=torch.float32, device=_DEV)


def _encode(x, pool_scale):
    """(codes uint8 [..., D], scales uint8 [..., D / 16]) of x [..., D]."""
    t = torch.nan_to_num(x.float() / _const(pool_scale), nan=0.0, posinf=math.inf, neginf=-math.inf)
    g = t.unflatten(-1, (-1, 16))
    s = (g.abs().amax(-1) / _const(6.0)).clamp(max=448.0).to(torch.float8_e4m3fn)
    sf = s.float().unsqueeze(-1)
    a = torch.where(sf > 0, g.abs() / sf, 0.0)
    # nearest level, ties to the even code
    c = ((a > 0.25).byte() + (a >= 0.75).byte() + (a > 1.25).byte() + (a >= 1.75).byte()
         + (a > 2.5).byte() + (a >= 3.5).byte() + (a > 5.0).byte())
    c = c | (torch.signbit(g).byte() << 3)
    return c.flatten(-2), s.view(torch.uint8)


def _values(codes, scales):
    """c * s in fp32 for codes [..., D] and scales [..., D / 16]."""
    levels = torch.tensor(_LEVELS + tuple(-v for v in _LEVELS), dtype=torch.float32, device=codes.device)
    c = torch.index_select(levels, 0, codes.reshape(-1).int()).view(codes.shape)
    s = scales.view(torch.float8_e4m3fn).float()
    return (c.unflatten(-1, (-1, 16)) * s.unsqueeze(-1)).flatten(-2)


def _pack(codes, scales, is_key):
    """Pool tiles uint8 [..., 9 D] of 16 tokens' codes [..., 16, D] and scales [..., 16, D / 16]."""
    if is_key:
        codes = codes.unflatten(-1, (-1, 4, 4)).transpose(-3, -2).flatten(-3)
    else:
        scales = scales.transpose(-2, -1)
    two = codes.unflatten(-1, (-1, 2))
    return torch.cat([(two[..., 0] | (two[..., 1] << 4)).flatten(-2), scales.flatten(-2)], dim=-1)


def _unpack(tiles, is_key):
    """(codes [..., 16, D], scales [..., 16, D / 16]) of pool tiles [..., 9 D]."""
    d = tiles.shape[-1] // 9
    two = tiles[..., :8 * d].unflatten(-1, (16, d // 2))
    codes = torch.stack([two & 15, two >> 4], dim=-1).flatten(-2)
    if is_key:
        codes = codes.unflatten(-1, (4, d // 16, 4)).transpose(-3, -2).flatten(-3)
        scales = tiles[..., 8 * d:].unflatten(-1, (16, d // 16))
    else:
        scales = tiles[..., 8 * d:].unflatten(-1, (d // 16, 16)).transpose(-2, -1)
    return codes, scales.contiguous()


# ── inputs ───────────────────────────────────────────────────────────────
def _pool(case, gen, blocks, dtype, drift):
    """One pool's rows [blocks, Hkv, page, D]: unit normal, keys with a part that a page has in common, as neighbouring tokens do."""
    x = torch.randn(blocks, case["heads"], case["page"], case["dim"], generator=gen, device=_DEV, dtype=dtype)
    if drift:
        x += 0.7 * torch.randn(blocks, case["heads"], 1, case["dim"], generator=gen, device=_DEV, dtype=dtype)
    return x


def _quantised(x, which, is_key):
    """The 4-bit pool of the rows x [blocks, Hkv, page, D], a slice of blocks at a time."""
    nb, hkv, page, dim = x.shape
    out = torch.empty(nb, hkv, page // 16, 9 * dim, dtype=torch.uint8, device=_DEV)
    step = max(1, (1 << 26) // (hkv * page * dim))
    out_parts, parts = out.split(step), x.split(step)
    list(map(lambda o, p: o.copy_(_pack(*_encode(p.unflatten(2, (-1, 16)), _SCALES[which]), is_key)), out_parts, parts))
    return out


def prepare(case, seed):
    gen = torch.Generator(device=_DEV).manual_seed(seed)
    heads, dim, page = case["heads"], case["dim"], case["page"]
    if case["op"] == "store":
        n = case["tokens"]
        width = 2 * heads * dim + case["pad"]
        rows = torch.randn(n, width, generator=gen, device=_DEV).half()
        blocks = -(-n // page) + 3
        # decode steps land in scattered slots, prompts in runs of a page
        slots = (torch.randperm(blocks, generator=gen, device=_DEV)[:, None] * page + torch.arange(page, device=_DEV)).flatten()[:n]
        if n <= 64:
            slots = slots[torch.randperm(n, generator=gen, device=_DEV)]
        if case["skip"]:
            slots[::case["skip"]] = -1
        pools = torch.zeros(2, blocks, heads, page // 16, 9 * dim, dtype=torch.uint8, device=_DEV)
        key = rows[:, :heads * dim].unflatten(1, (heads, dim))
        value = rows[:, heads * dim:2 * heads * dim].unflatten(1, (heads, dim))
        return dict(case=case, key=key, value=value, slots=slots, kc=pools[0], vc=pools[1])

    lens = _lens(case, seed)
    pages = -(-lens // page)
    # the summaries come back whole, so their pool has one size for every seed
    blocks = case["seqs"] * -(-case["high"] // page) + 2 if case["op"] == "bounds" else int(pages.sum() * 1.1) + 2
    rng = np.random.default_rng(seed + 1)
    ids = rng.permutation(blocks)[:pages.sum()]
    table = np.full((case["seqs"], max(1, int(pages.max()))), -1, dtype=np.int32)
    table[np.arange(table.shape[1])[None] < pages[:, None]] = ids
    st = dict(case=case, table=torch.from_numpy(table).to(_DEV), lens=torch.from_numpy(lens.astype(np.int32)).to(_DEV))
    dtype = torch.float32 if case.get("fp32") else torch.float16
    k = _pool(case, gen, blocks, dtype, True)
    if case["op"] == "bounds":
        st["kc"] = k
        st["bounds"] = torch.zeros(blocks, heads, 2, dim, dtype=dtype, device=_DEV)
        return st
    v = _pool(case, gen, blocks, dtype, False)
    st["q"] = torch.randn(case["seqs"], case["q_heads"], dim, generator=gen, device=_DEV, dtype=dtype)
    q4 = case["op"] == "q4" or case["q4"]
    st["kc"], st["vc"] = (_quantised(k, "k", True), _quantised(v, "v", False)) if q4 else (k, v)
    if case["op"] == "sparse":
        # the summaries a program keeps beside its pools, of the keys as the cache holds them, valid tokens only
        if q4:
            k = _read_pool(st["kc"], "k", True)
        last = (lens - 1) // page
        some = lens > 0
        tail = np.full(blocks, page)
        tail[table[np.nonzero(some)[0], last[some]]] = lens[some] - last[some] * page
        live = (torch.arange(page, device=_DEV) < torch.from_numpy(tail).to(_DEV)[:, None])[:, None, :, None]
        big = torch.finfo(dtype).max
        st["bounds"] = torch.stack([torch.where(live, k, big).amin(2), torch.where(live, k, -big).amax(2)], dim=2)
    return st


# ── plain forms ──────────────────────────────────────────────────────────
def _read_pool(pool, which, is_key):
    """A whole 4-bit pool as fp16 rows [blocks, Hkv, page, D]."""
    return (_values(*_unpack(pool, is_key)) * _const(_SCALES[which])).half().flatten(2, 3)


def _plain_store(st):
    live = (st["slots"] >= 0)[:, None, None]
    return tuple(torch.where(live, _values(*_encode(st[x], _SCALES[w])) * _const(_SCALES[w]), 0.0).half() for x, w in (("key", "k"), ("value", "v")))


def _softmax_av(q, k, v, live, scale):
    """q [..., G, D], k and v [..., L, D], live [..., L] -> [..., G, D] in fp32; rows with nothing live are 0."""
    s = (q @ k.transpose(-2, -1)) * scale
    s = torch.where(live.unsqueeze(-2), s, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    return (p @ v) / torch.where(total == 0, 1.0, total)


def _plain_q4(st):
    case, q = st["case"], st["q"]
    b, page, dim = case["seqs"], case["page"], case["dim"]
    at = st["table"].clamp(min=0).long()
    # [B, pages, Hkv, page / 16, 16, D] -> [B, Hkv, tokens, D]
    k = _values(*_unpack(st["kc"][at], True)).flatten(3, 4).transpose(1, 2).flatten(2, 3)
    v = _values(*_unpack(st["vc"][at], False)).flatten(3, 4).transpose(1, 2).flatten(2, 3)
    live = (torch.arange(k.shape[2], device=_DEV) < st["lens"][:, None])[:, None]
    qg = q.float().view(b, case["heads"], -1, dim)
    out = _softmax_av(qg, k, v, live, _SCALES["k"] / math.sqrt(dim))
    return (out * _SCALES["v"]).half().view(q.shape)


def _plain_bounds(st):
    case, kc, bounds = st["case"], st["kc"], st["bounds"]
    page, new = case["page"], case["new"]
    lens = st["lens"].long()
    pages = (lens + page - 1) // page
    first = (lens - new).clamp(min=0) // page if new else torch.zeros_like(lens)
    at = torch.arange(st["table"].shape[1], device=_DEV)
    due = (at >= first[:, None]) & (at < pages[:, None])
    ids = st["table"][due].long()
    left = (lens[:, None] - at * page)[due]
    live = (torch.arange(page, device=_DEV) < left[:, None])[:, None, :, None]
    big = torch.finfo(kc.dtype).max
    k = torch.nan_to_num(kc[ids], nan=0.0, posinf=big, neginf=-big)
    bounds[ids] = torch.stack([torch.where(live, k, big).amin(2), torch.where(live, k, -big).amax(2)], dim=2)
    return bounds


def _plain_select(st):
    """Kept pages [B, Hkv, keep], ascending, -1 past the last. Scores in 64 bits: near ties decide which page is kept."""
    case = st["case"]
    b, heads, dim, page, keep = case["seqs"], case["heads"], case["dim"], case["page"], case["keep"]
    bounds = st["bounds"][st["table"].clamp(min=0).long()].transpose(1, 2)  # [B, Hkv, P, 2, D]
    q = st["q"].view(b, heads, -1, dim).double()
    score = q.clamp(min=0) @ bounds[..., 1, :].double().transpose(-2, -1) + q.clamp(max=0) @ bounds[..., 0, :].double().transpose(-2, -1)
    score = score.amax(2)
    at = torch.arange(score.shape[-1], device=_DEV)
    pages = ((st["lens"].long() + page - 1) // page)[:, None, None]
    score = torch.where((at < case["sink"]) | (at >= pages - case["recent"]), math.inf, score)
    score = torch.where(at < pages, score, -math.inf)
    order = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :keep]
    order = torch.where(order < pages, order, 1 << 30).sort(-1).values
    kept = torch.where(order < (1 << 30), order, -1)
    return torch.nn.functional.pad(kept, (0, keep - kept.shape[-1]), value=-1)


def _plain_sparse(st):
    case, q = st["case"], st["q"]
    b, heads, dim, page = case["seqs"], case["heads"], case["dim"], case["page"]
    kept = _plain_select(st)
    row = torch.arange(b, device=_DEV)[:, None, None]
    head = torch.arange(heads, device=_DEV)[:, None]
    ids = st["table"][row, kept.clamp(min=0)].clamp(min=0).long()
    if case["q4"]:
        k = _values(*_unpack(st["kc"][ids, head], True)).flatten(2, 4)
        v = _values(*_unpack(st["vc"][ids, head], False)).flatten(2, 4)
        ks, vs = _SCALES["k"], _SCALES["v"]
    else:
        k, v = st["kc"][ids, head].float().flatten(2, 3), st["vc"][ids, head].float().flatten(2, 3)
        ks, vs = 1.0, 1.0
    token = (kept.unsqueeze(-1) * page + torch.arange(page, device=_DEV)).flatten(2)
    live = (token >= 0) & (kept >= 0).repeat_interleave(page, -1) & (token < st["lens"].long()[:, None, None])
    out = _softmax_av(q.float().view(b, heads, -1, dim), k, v, live, ks / math.sqrt(dim))
    return dict(out=(out * vs).to(q.dtype).view(q.shape), kept=kept.int())


# ── one pass ─────────────────────────────────────────────────────────────
def run(st):
    case = st["case"]
    if not own:
        return {"store": _plain_store, "q4": _plain_q4, "bounds": _plain_bounds, "sparse": _plain_sparse}[case["op"]](st)
    from xllms_b200 import operator_api as pa
    scales = (_SCALES["k"], _SCALES["v"])
    if case["op"] == "store":
        pa.reshape_and_cache_q4(st["key"], st["value"], st["kc"], st["vc"], st["slots"], *scales)
        return pa.read_cache_q4(st["kc"], st["vc"], st["slots"], *scales)
    if case["op"] == "q4":
        return pa.paged_attention_q4(st["q"], st["kc"], st["vc"], st["table"], st["lens"], *scales)
    if case["op"] == "bounds":
        return pa.page_bounds(st["kc"], st["table"], st["lens"], st["bounds"], num_new_tokens=case["new"])
    kept = torch.empty(case["seqs"], case["heads"], case["keep"], dtype=torch.int32, device=_DEV)
    kind = dict(k_scale=scales[0], v_scale=scales[1]) if case["q4"] else {}
    out = pa.paged_attention_sparse(st["q"], st["kc"], st["vc"], st["bounds"], st["table"], st["lens"], case["keep"], sink_pages=case["sink"],
                                    recent_pages=case["recent"], selected=kept, **kind)
    return dict(out=out, kept=kept)


def work(case):
    """Each input read once, each output written once; lengths at the middle of their range."""
    heads, dim = case["heads"], case["dim"]
    row4 = dim * 9 / 16
    if case["op"] == "store":
        n = case["tokens"] * (1 - (1 / case["skip"] if case["skip"] else 0))
        # fp16 rows in, 4-bit rows out; 4-bit rows in, fp16 rows out
        return dict(bytes=2 * n * heads * (2 * dim + 2 * row4) + 2 * (case["tokens"] - n) * heads * 2 * dim + 16 * case["tokens"], flops=10 * n * heads * dim)
    es = 4 if case.get("fp32") else 2
    tokens = case["seqs"] * (case["low"] + case["high"]) / 2
    pages = tokens / case["page"]
    if case["op"] == "bounds":
        new = min(tokens, case["seqs"] * case["new"]) if case["new"] else tokens
        return dict(bytes=new * heads * dim * es + max(case["seqs"], new / case["page"]) * heads * 2 * dim * es, flops=2 * new * heads * dim)
    io = 2 * case["seqs"] * case["q_heads"] * dim * es + 4 * pages + 4 * case["seqs"]
    if case["op"] == "q4":
        return dict(bytes=tokens * heads * 2 * row4 + io, flops=4 * tokens * case["q_heads"] * dim)
    kept = min(tokens, case["seqs"] * case["keep"] * case["page"])
    scored = pages if pages > case["seqs"] * case["keep"] else 0
    row = row4 if case["q4"] else dim * es
    return dict(bytes=scored * heads * 2 * dim * es + kept * heads * 2 * row + io + 4 * case["seqs"] * heads * case["keep"],
                flops=4 * (kept + scored) * case["q_heads"] * dim)


# ── the same in 64 bits, from the definitions ────────────────────────────
def _exact_store(x, pool_scale):
    t = np.nan_to_num((x.float().cpu().numpy() / np.float32(pool_scale)).astype(np.float64), nan=0.0, posinf=np.inf, neginf=-np.inf)
    t = t.reshape(t.shape[:-1] + (-1, 16))
    amax = np.abs(t).max(-1, keepdims=True) / 6
    step = np.exp2(np.maximum(np.floor(np.log2(np.maximum(amax, 1e-30))), -6) - 3)
    s = np.minimum(np.rint(amax / step) * step, 448.0)
    y = np.divide(np.abs(t), s, out=np.zeros_like(t), where=s > 0)
    fine = np.where(y < 2, 0.5, np.where(y < 4, 1.0, 2.0))
    c = np.minimum(np.rint(y / fine) * fine, 6.0)
    return (np.copysign(c, t) * s * np.float64(np.float32(pool_scale))).reshape(x.shape)


def _exact_rows(pool, which, is_key, at, heads):
    """Rows in fp64 [Hkv, tokens, D] of one sequence's pages `at`, byte by byte."""
    if pool.dtype != torch.uint8:
        return pool[at].double().permute(1, 0, 2, 3).flatten(1, 2)
    tile = pool[at].permute(1, 0, 2, 3).flatten(1, 2)  # [Hkv, pages * page / 16, 9 D]
    d = tile.shape[-1] // 9
    ch = torch.arange(d, device=_DEV)
    tok = torch.arange(16, device=_DEV)[:, None]
    if is_key:
        nib = tok * d + (ch % 16) // 4 * (d // 4) + ch // 16 * 4 + ch % 4
        sc = 8 * d + tok * (d // 16) + ch // 16
    else:
        nib = tok * d + ch
        sc = 8 * d + ch // 16 * 16 + tok
    code = (tile[..., nib // 2] >> ((nib % 2) * 4).byte()) & 15
    e, m = (code >> 1) & 3, (code & 1).double()
    mag = torch.where(e == 0, 0.5 * m, (1 + 0.5 * m) * torch.exp2(e.double() - 1))
    b = tile[..., sc]
    se, sm = ((b >> 3) & 15).double(), (b & 7).double()
    s = torch.where(se == 0, sm / 8 * 2.0 ** -6, (1 + sm / 8) * torch.exp2(se - 7))
    return (torch.where(code > 7, -mag, mag) * s * float(np.float32(_SCALES[which]))).flatten(1, 2)


def _exact_attention(q, k, v):
    """q [Hq, D], k and v [Hkv, L, D] -> [Hq, D]."""
    s = torch.einsum("hgd,hld->hgl", q.unflatten(0, (k.shape[0], -1)), k) / math.sqrt(q.shape[-1])
    return torch.einsum("hgl,hld->hgd", torch.softmax(s, -1), v).flatten(0, 1)


def exact(case, seed):
    st = prepare(case, seed)
    heads, page = case["heads"], case["page"]
    if case["op"] == "store":
        dead = (st["slots"] < 0).cpu().numpy()
        got = [_exact_store(st["key"], _SCALES["k"]), _exact_store(st["value"], _SCALES["v"])]
        for x in got:
            x[dead] = 0
        return tuple(got)
    table, lens = st["table"], st["lens"].tolist()
    if case["op"] == "bounds":
        want = st["bounds"].double()
        big = float(torch.finfo(st["kc"].dtype).max)
        for b, n in enumerate(lens):
            pages = -(-n // page)
            lo = max(0, n - case["new"]) // page if case["new"] else 0
            if lo == pages:
                continue
            x = torch.nan_to_num(st["kc"][table[b, lo:pages].long()].double(), nan=0.0, posinf=big, neginf=-big)
            whole = torch.stack([x.amin(2), x.amax(2)], 2)
            end = x[-1, :, :n - (pages - 1) * page]
            whole[-1] = torch.stack([end.amin(1), end.amax(1)], 1)
            want[table[b, lo:pages].long()] = whole
        return want
    q = st["q"].double()
    out = torch.zeros_like(q)
    if case["op"] == "q4":
        for b, n in enumerate(lens):
            if n:
                at = table[b, :-(-n // page)].long()
                out[b] = _exact_attention(q[b], *(_exact_rows(st[p], w, w == "k", at, heads)[:, :n] for p, w in (("kc", "k"), ("vc", "v"))))
        return out
    keep = case["keep"]
    group = case["q_heads"] // heads
    for b, n in enumerate(lens):
        pages = -(-n // page)
        if not n:
            continue
        at = table[b, :pages].long()
        bd = st["bounds"][at].double()  # [P, Hkv, 2, D]
        for h in range(heads):
            qh = q[b, h * group:(h + 1) * group]
            chosen = list(range(pages))
            if pages > keep:
                # one query head at a time, so that the terms fit
                sc = torch.stack([torch.maximum(qh[g] * bd[:, h, 0], qh[g] * bd[:, h, 1]).sum(-1) for g in range(group)]).amax(0).cpu().numpy()
                must = set(range(case["sink"])) | set(range(pages - case["recent"], pages))
                rest = [p for p in np.argsort(-sc, kind="stable") if p not in must]
                chosen = sorted(must | set(int(p) for p in rest[:keep - len(must)]))
            rows = [_exact_rows(st[p][:, h:h + 1], w, w == "k", at[chosen], 1) for p, w in (("kc", "k"), ("vc", "v"))]
            total = (len(chosen) - 1) * page + n - (pages - 1) * page
            out[b, h * group:(h + 1) * group] = _exact_attention(qh, *(x[:, :total] for x in rows))
    return dict(out=out, kept=None)
