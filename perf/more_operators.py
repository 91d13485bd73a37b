"""Performance cases of a serving step on a paged KV cache whose pages are handed out on the GPU, held in 8
bits with a scale for each block of 16 positions and head, and attended whole or by selected pages.

Kinds:

  assign   pages of the pool handed to the sequences that grow, taken back from those that end; positions,
           lengths, offsets and the new tokens' slots for the operators after it
  append   keys and values of new tokens stored as e4m3 under scales of their blocks of 16 positions, which
           grow with the values, with the position rotation of q and k on the way
  decode   attention of one new token per sequence over such a cache
  bounds   the smallest and largest key of every page that new tokens complete, dim by dim
  sparse   attention of one new token per sequence over the pages of each that a score selects: the largest
           scalar product that a page's bounds allow with the query

Head counts are those of perf/cases.py's models (40 / 8, 16 / 4 and 32 / 8 heads of 128).  Activations are
N(0, 1), stored keys and values too, times a size of their KV head.  Pages are scattered over the pool as
after some time of serving.
"""
import math

import torch

own = False

DEV = "cuda:0"
D = 128
BLOCK = 16
E4M3_MAX = 448.0
LEAST = 2.0 ** -126
HEADS = {"h3136": (40, 8), "h2048": (16, 4), "h2560": (32, 8)}


def listed():
    return [
        # a decode step of a large serving batch: every 64th sequence or so needs a page, some have ended
        {"name": "assign_256_tokens", "kind": "assign", "page": 64, "batch": 256, "shortest": 1, "longest": 1,
         "start": 8000, "ended": 9, "idle": 20, "spare": 40},
        # prompts that enter beside them, more than the pool has pages for
        {"name": "assign_60_prompts", "kind": "assign", "page": 16, "batch": 60, "shortest": 3, "longest": 900,
         "start": 0, "ended": 0, "idle": 0, "spare": 800},
        # a decode step of a serving batch, partial rotation of neighbouring pairs
        {"name": "append_24_tokens", "kind": "append", "model": "h2560", "page": 32, "batch": 24, "shortest": 1,
         "longest": 1, "start": 30000, "rotary": 64, "interleaved": True},
        # further turns of running conversations, a model without rotation: keys and values only
        {"name": "append_5_prompts", "kind": "append", "model": "h2048", "page": 64, "batch": 5, "shortest": 61,
         "longest": 1801, "start": 700, "rotary": 0, "interleaved": False},
        # one long document, its rotated q and k returned for the attention over it
        {"name": "append_long_prompt", "kind": "append", "model": "h3136", "page": 128, "batch": 1, "shortest": 8191,
         "longest": 8191, "start": 0, "rotary": 128, "interleaved": False},
        # one conversation: a call that latency bounds
        {"name": "decode_1x1300", "kind": "decode", "model": "h3136", "page": 16, "batch": 1, "shortest": 1300,
         "longest": 1300, "idle": 0},
        # a serving batch, in a step captured for more sequences than are active
        {"name": "decode_90_chats", "kind": "decode", "model": "h2560", "page": 32, "batch": 90, "shortest": 40,
         "longest": 5000, "idle": 6},
        # a book beside a new conversation
        {"name": "decode_long", "kind": "decode", "model": "h3136", "page": 128, "batch": 2, "shortest": 33,
         "longest": 90001, "idle": 0},
        # the decode step's: few of its tokens complete a page
        {"name": "bounds_100_tokens", "kind": "bounds", "model": "h3136", "cache": "block", "page": 16, "batch": 100,
         "shortest": 1, "longest": 1, "start": 5000},
        # prompts of a bf16 cache
        {"name": "bounds_3_prompts", "kind": "bounds", "model": "h2048", "cache": "bf16", "page": 64, "batch": 3,
         "shortest": 700, "longest": 9000, "start": 20},
        # one long conversation, 2048 positions of 100000 attended
        {"name": "sparse_1x100001", "kind": "sparse", "model": "h3136", "cache": "block", "page": 64, "batch": 1,
         "shortest": 100001, "longest": 100001, "select": 32, "idle": 0},
        # a batch of documents of which some are shorter than what is attended
        {"name": "sparse_20_documents", "kind": "sparse", "model": "h2560", "cache": "bf16", "page": 32, "batch": 20,
         "shortest": 900, "longest": 30000, "select": 63, "idle": 2},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["assign", "append", "decode", "bounds", "sparse"])
    case = {"kind": kind, "page": rng.choice([16, 32, 64, 128, 256])}
    if kind == "assign":
        case["batch"] = _log(rng, 1, 500)
        prompts = rng.random() < 0.5
        case["longest"] = _log(rng, 2, max(2, 16000 // case["batch"])) if prompts else 1
        case["shortest"] = rng.randint(1, case["longest"])
        case["start"] = rng.choice([0, _log(rng, 1, 8000)])
        case["ended"] = rng.randint(0, case["batch"] // 4)
        case["idle"] = rng.randint(0, case["batch"] // 4)
        case["spare"] = _log(rng, 1, 2 * case["batch"] * (1 + case["longest"] // case["page"]))
        return case
    case["model"] = rng.choice(["h3136", "h2048", "h2560"])
    case["batch"] = _log(rng, 1, 64)
    if kind in ("append", "bounds"):
        prompts = rng.random() < 0.5
        case["longest"] = _log(rng, 2, 8192 // case["batch"]) if prompts else 1
        case["shortest"] = rng.randint(1, case["longest"])
        case["start"] = rng.choice([0, _log(rng, 1, 60000)]) if prompts else _log(rng, 1, 60000)
        if kind == "append":
            case["rotary"] = rng.choice([0, 32, 64, 96, 128, 128])
            case["interleaved"] = rng.random() < 0.5
        else:
            case["cache"] = rng.choice(["bf16", "e4m3", "block"])
        return case
    case["longest"] = _log(rng, 1, min(60000, 160000 // case["batch"]))
    case["shortest"] = _log(rng, 1, case["longest"]) if case["longest"] > 1 else 1
    case["idle"] = rng.choice([0, 0, rng.randint(0, case["batch"] - 1)])
    if kind == "sparse":
        case["cache"] = rng.choice(["bf16", "e4m3", "block"])
        case["select"] = _log(rng, 1, 100)
    return case


def _lengths(case):
    """The sequences' lengths, from the longest to the shortest over their logarithm, in scattered order."""
    n, lo, hi = case["batch"], case["shortest"], case["longest"]
    step = next(s for s in (7, 5, 3, 1) if math.gcd(s, n) == 1)
    lens = [int(round(hi * (lo / hi) ** ((step * i % n) / max(1, n - 1)))) for i in range(n)]
    if case["kind"] != "assign":
        for i in range(case.get("idle", 0)):
            lens[n - 1 - i] = 0
    return lens


def _starts(case):
    """Positions stored before the call: no two alike, 0 where the case begins with nothing."""
    if not case["start"]:
        return [0] * case["batch"]
    if case["kind"] == "assign":
        return [(case["start"] * (i + 1) // case["batch"] + 37 * i) % (case["start"] + 1) for i in range(case["batch"])]
    return [case["start"] + 37 * i for i in range(case["batch"])]


def _roles(case):
    """New tokens per sequence of an assignment: -1 where it has ended, 0 where it waits."""
    new = _lengths(case)
    for i in range(case["ended"]):
        new[4 * i] = -1
    for i in range(case["idle"]):
        new[4 * i + 1 if 4 * i + 1 < len(new) else 0] = 0
    return new


# --- inputs ---------------------------------------------------------------------------------


def _normal(gen, *shape):
    return torch.randn(shape, generator=gen, device=DEV)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _cumulative(lens):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return at


def _power_of_two(amax):
    """The smallest power of two s, 2^-126 at least, with amax <= 448 s."""
    f, e = torch.frexp(amax.double().clamp_min(LEAST) / E4M3_MAX)   # in [0.5, 1): powers of two are 0.5
    return torch.ldexp(torch.ones_like(f), e - (f == 0.5).int()).clamp_min(LEAST).float()


def _e4m3(x):
    return x.clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)


def _pool(case, gen, n_pages, n_kv, cache):
    """K and V pages [n_pages, n_kv, page, 128] that hold earlier tokens, and their scales (None: bf16)."""
    size = torch.exp2(4 * torch.rand(2, n_kv, 1, 1, generator=gen, device=DEV) - 2)
    pages = [_normal(gen, n_pages, n_kv, case["page"], D) * size[i] for i in range(2)]
    if cache == "bf16":
        return [p.to(torch.bfloat16) for p in pages], [None, None]
    if cache == "e4m3":
        scales = [size[i, :, 0, 0] * 0.01 for i in range(2)]
        return [_e4m3(p / s[:, None, None]) for p, s in zip(pages, scales)], scales
    held, scales = [], []
    for p in pages:
        blocks = p.view(n_pages, n_kv, -1, BLOCK * D)
        s = _power_of_two(blocks.abs().amax(-1))
        held.append(_e4m3(blocks / s[..., None]).view(p.shape))
        scales.append(s)
    return held, scales


def _bounds_of(state):
    """The bounds of every page of the pool."""
    k = _values(state["k_pages"], state["k_scale"])
    return torch.stack((k.amin(2), k.amax(2)), dim=2).to(torch.bfloat16).contiguous()


def _prepare_assign(case, gen):
    lens, new, page = _starts(case), _roles(case), case["page"]
    decode = case["longest"] == 1
    have = [-(-n // page) for n in lens]
    width = max(1, max(-(-(n + max(0, m)) // page) for n, m in zip(lens, new))) + 1
    n_pages = sum(have) + case["spare"] + 5000                           # (the last of other batches)
    order = torch.randperm(n_pages, generator=gen, device=DEV).to(torch.int32)
    used = torch.arange(width, device=DEV)[None] < _ints(have)[:, None]
    table = torch.full((case["batch"], width), -1, dtype=torch.int32, device=DEV)
    table[used] = order[:sum(have)]
    free = torch.full((n_pages,), -1, dtype=torch.int32, device=DEV)
    free[:case["spare"]] = order[sum(have):sum(have) + case["spare"]]
    return {"case": dict(case), "lens": _ints(lens), "new_lens": _ints(new), "page_table": table, "free_pages": free,
            "free_count": _ints([case["spare"]]), "decode": decode,
            "tokens": None if decode else sum(max(0, m) for m in new)}


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    if case["kind"] == "assign":
        return _prepare_assign(case, gen)
    H, n_kv = HEADS[case["model"]]
    lens, page = _lengths(case), case["page"]
    state = {"case": dict(case), "H": H, "n_kv": n_kv}
    if case["kind"] in ("decode", "sparse"):
        counts = [-(-n // page) for n in lens]
        n_pages = max(1, sum(counts))
        (state["k_pages"], state["v_pages"]), (state["k_scale"], state["v_scale"]) = \
            _pool(case, gen, n_pages, n_kv, case.get("cache", "block"))
        # every sequence's pages, scattered over the pool; the entries after its last page are not in use
        order = torch.randperm(n_pages, generator=gen, device=DEV).to(torch.int32)
        width = max(1, max(counts))
        used = torch.arange(width, device=DEV)[None] < _ints(counts)[:, None]
        state["page_table"] = torch.full((case["batch"], width), -1, dtype=torch.int32, device=DEV)
        state["page_table"][used] = order[:sum(counts)]
        state["kv_lens"] = _ints(lens)
        state["q"] = _normal(gen, case["batch"], H * D).to(torch.bfloat16)
        if case["kind"] == "sparse":
            state["k_bounds"] = _bounds_of(state)
        return state
    T, starts = sum(lens), _starts(case)
    # the pages of the new tokens are each sequence's own
    spans = [(s // page, -(-(s + n) // page)) for s, n in zip(starts, lens)]
    n_pages = sum(b - a for a, b in spans) + 3
    (state["k_pages"], state["v_pages"]), (state["k_scale"], state["v_scale"]) = \
        _pool(case, gen, n_pages, n_kv, case.get("cache", "block"))
    order = torch.randperm(n_pages, generator=gen, device=DEV).to(torch.int32)
    rows = torch.full((case["batch"], max(b for _, b in spans)), int(order[-1]), dtype=torch.int32)
    at, ids = 0, order.cpu()
    for i, (a, b) in enumerate(spans):
        rows[i, a:b] = ids[at:at + b - a]
        at += b - a
    state["page_table"] = rows.to(DEV)
    state["start_pos"] = _ints(starts)
    state["decode"] = case["longest"] == 1
    state["tokens"] = T
    state["cu_seqlens"] = None if state["decode"] else _ints(_cumulative(lens))
    if case["kind"] == "bounds":
        state["k_bounds"] = _normal(gen, n_pages, n_kv, 2, D).to(torch.bfloat16)     # of the pages' earlier owners
        return state
    qkv = _normal(gen, T, (H + 2 * n_kv) * D).to(torch.bfloat16)       # as one projection writes them
    state["q"], state["k"], state["v"] = qkv[:, :H * D], qkv[:, H * D:(H + n_kv) * D], qkv[:, (H + n_kv) * D:]
    state["inv_freq"] = None
    if case["rotary"]:
        state["inv_freq"] = 10000.0 ** (-torch.arange(0, case["rotary"], 2, device=DEV, dtype=torch.float32) / case["rotary"])
    return state


# --- one pass -------------------------------------------------------------------------------


def run(state):
    if own:
        return _run_own(state)
    return {"assign": _assign, "append": _append, "decode": _decode, "bounds": _bounds,
            "sparse": _sparse}[state["case"]["kind"]](state)


def _run_own(s):
    from nemotron_infer_amd import ops

    kind = s["case"]["kind"]
    if kind == "assign":
        step = ops.kv_assign_paged(s["lens"], s["new_lens"], s["page_table"], s["free_pages"], s["free_count"],
                                   s["case"]["page"], tokens=s["tokens"])
        return {**step._asdict(), "page_table": s["page_table"], "free_pages": s["free_pages"]}
    if kind == "decode":
        return ops.sdpa_decode_paged(s["q"], s["k_pages"], s["v_pages"], s["page_table"], s["kv_lens"],
                                     k_scale=s["k_scale"], v_scale=s["v_scale"])
    if kind == "sparse":
        return ops.sdpa_decode_paged_sparse(s["q"], s["k_pages"], s["v_pages"], s["page_table"], s["kv_lens"],
                                            s["k_bounds"], s["case"]["select"], k_scale=s["k_scale"], v_scale=s["v_scale"])
    if kind == "bounds":
        return ops.kv_bounds_paged(s["k_pages"], s["page_table"], s["start_pos"], s["k_bounds"], cu_seqlens=s["cu_seqlens"],
                                   tokens=None if s["decode"] else s["tokens"], k_scale=s["k_scale"])
    rotate = s["inv_freq"] is not None
    # a decode step needs no k of its own afterwards: the attention reads the cache
    k_out = torch.empty(s["k"].shape, dtype=torch.bfloat16, device=DEV) if rotate and not s["decode"] else None
    q_out, k_out = ops.kv_append_paged(s["k"], s["v"], s["k_pages"], s["v_pages"], s["page_table"], s["start_pos"],
                                       cu_seqlens=s["cu_seqlens"], q=s["q"] if rotate else None, inv_freq=s["inv_freq"],
                                       interleaved=s["case"]["interleaved"], k_scale=s["k_scale"], v_scale=s["v_scale"],
                                       k_out=k_out)
    return {"q": q_out, "k": k_out, "k_pages": s["k_pages"], "v_pages": s["v_pages"], "k_scale": s["k_scale"],
            "v_scale": s["v_scale"]}


def _assign(s):
    page, table, free = s["case"]["page"], s["page_table"], s["free_pages"]
    lens, new, count = s["lens"].long(), s["new_lens"].long(), s["free_count"].long()
    j = torch.arange(table.shape[1], device=DEV)[None]
    used, ended = -(-lens.clamp_min(0) // page), (lens >= 0) & (new < 0)
    # pages of the sequences that ended, pushed
    back = torch.where(ended, used, 0)
    mine = j < back[:, None]
    free[(count + (back.cumsum(0) - back)[:, None] + j)[mine]] = table[mine]
    count = count + back.sum()
    # pages for the new tokens, popped
    n = torch.where((lens >= 0) & (new > 0), new, 0)
    fits = lens + n <= table.shape[1] * page
    need = torch.where((n > 0) & fits, -(-(lens + n).clamp_min(0) // page) - used, 0)
    upto = need.cumsum(0)
    granted = (n > 0) & fits & ((need == 0) | (upto <= count))
    taken = torch.where(granted, need, 0)
    mine = (j >= used[:, None]) & (j < (used + taken)[:, None])
    table[mine] = free[(count - 1 - ((upto - need)[:, None] + j - used[:, None]))[mine]]
    start = torch.where(granted, lens, -1)
    after = torch.where(ended, -1, torch.where(granted, lens + n, lens))
    # the new tokens' places in the pool
    if s["decode"]:
        cu = None
        row, place = torch.arange(len(lens), device=DEV), torch.zeros(len(lens), dtype=torch.int64, device=DEV)
    else:
        cu = torch.cat((torch.zeros(1, dtype=torch.int64, device=DEV), new.clamp_min(0).cumsum(0)))
        t = torch.arange(s["tokens"], device=DEV)
        row = torch.searchsorted(cu[1:], t, right=True)
        place = t - cu[row]
    pos = (start[row] + place).clamp_min(0)
    slots = torch.where(start[row] >= 0, table[row, (pos // page).clamp_max(table.shape[1] - 1)].long() * page + pos % page, -1)
    return {"start_pos": start.int(), "kv_lens": torch.where(granted, lens + n, 0).int(),
            "cu_seqlens": None if cu is None else cu.int(), "slots": slots, "lens": after.int(),
            "free_count": (count - taken.sum()).int(), "page_table": table, "free_pages": free}


def _tokens(s):
    """Sequence and place in it of every packed token."""
    t = torch.arange(s["tokens"], device=DEV)
    if s["decode"]:
        return t, torch.zeros_like(t)
    cu = s["cu_seqlens"].long()
    b = torch.searchsorted(cu[1:], t, right=True)
    return b, t - cu[b]


def _rotate(x, cos, sin, interleaved):
    """x [T, heads, 128]; cos, sin [T, 1, rotary / 2]."""
    half = cos.shape[-1]
    turned = x[..., :2 * half]
    a, b = (turned[..., 0::2], turned[..., 1::2]) if interleaved else (turned[..., :half], turned[..., half:])
    pair = (a * cos - b * sin, a * sin + b * cos)
    turned = torch.stack(pair, dim=-1).flatten(-2) if interleaved else torch.cat(pair, dim=-1)
    return torch.cat((turned, x[..., 2 * half:]), dim=-1)


def _append(s):
    case, T, n_kv, page = s["case"], s["tokens"], s["n_kv"], s["case"]["page"]
    b, place = _tokens(s)
    pos = s["start_pos"].long()[b] + place
    k, v = (s[n].float().view(T, n_kv, D) for n in ("k", "v"))
    q_out = k_out = None
    if s["inv_freq"] is not None:
        angle = pos.double()[:, None] * s["inv_freq"].double()
        cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
        q_out = _rotate(s["q"].float().view(T, s["H"], D), cos, sin, case["interleaved"]).to(torch.bfloat16).view(T, -1)
        # (in 64 bits: the largest of a block decides its scale, which is a power of two)
        k = _rotate(k.double(), cos.double(), sin.double(), case["interleaved"]).float()
        if not s["decode"]:
            k_out = k.to(torch.bfloat16).view(T, -1)
    ids = s["page_table"].long()[b, pos // page]
    block = ids * (page // BLOCK) + pos % page // BLOCK                  # of the pool: one of each 16 positions
    n_blocks = s["k_pages"].shape[0] * (page // BLOCK)
    # the first place that a block's new tokens take: what lies before it was stored earlier
    first = torch.full((n_blocks,), BLOCK, dtype=torch.int64, device=DEV).scatter_reduce(0, block, pos % BLOCK, "amin")
    touched = torch.nonzero(first < BLOCK)[:, 0]
    page_of, part = touched // (page // BLOCK), touched % (page // BLOCK)
    old = (first[touched] > 0)[:, None]
    rows = part[:, None] * BLOCK + torch.arange(BLOCK, device=DEV)
    earlier = torch.arange(BLOCK, device=DEV)[None] < first[touched][:, None]
    for pages, scales, x in ((s["k_pages"], s["k_scale"], k), (s["v_pages"], s["v_scale"], v)):
        amax = torch.zeros(n_blocks, n_kv, device=DEV)
        amax = amax.scatter_reduce(0, block[:, None].expand(T, n_kv), x.abs().amax(-1), "amax")[touched]
        was = scales[page_of, :, part]
        s_new = torch.maximum(_power_of_two(amax), torch.where(old, was, torch.zeros_like(was)))
        codes = pages.view(torch.uint8)
        held = codes[page_of[:, None], :, rows].view(pages.dtype).float()            # [blocks, 16, n_kv, 128]
        moved = _e4m3(held * (was / s_new)[:, None, :, None]).view(torch.uint8)
        grown = earlier[:, :, None] & (s_new > was)[:, None]
        at, r, h = torch.nonzero(grown, as_tuple=True)
        codes[page_of[at], h, rows[at, r]] = moved[at, r, h]
        scales[page_of, :, part] = s_new
        codes[ids, :, pos % page] = _e4m3(x / scales[ids, :, pos % page // BLOCK][..., None]).view(torch.uint8)
    return {"q": q_out, "k": k_out, "k_pages": s["k_pages"], "v_pages": s["v_pages"], "k_scale": s["k_scale"],
            "v_scale": s["v_scale"]}


def _values(pages, scale):
    """What pages [n, n_kv, page, 128] stand for."""
    if scale is None:
        return pages.float()
    if scale.dim() == 1:
        return pages.float() * scale[:, None, None]
    n, n_kv = scale.shape[:2]
    return (pages.float().view(n, n_kv, -1, BLOCK, D) * scale[..., None, None]).view(n, n_kv, -1, D)


def _softmax(scores, mask):
    """Weights of the last axis where mask is true; a row without any gets zeros."""
    scores = scores.masked_fill(~mask, float("-inf"))
    top = scores.amax(dim=-1, keepdim=True).clamp_min(torch.finfo(scores.dtype).min)
    weights = (scores - top).exp()
    return weights / weights.sum(dim=-1, keepdim=True).clamp_min(torch.finfo(scores.dtype).tiny)


def _take(pages, scale, ids):
    """Pages `ids` [...] as [..., n_kv, page, 128] float32."""
    held = pages.view(torch.uint8)[ids].view(pages.dtype) if pages.dtype == torch.float8_e4m3fn else pages[ids]
    held = held.float()
    if scale is None:
        return held
    if scale.dim() == 1:
        return held * scale[:, None, None]
    return (held.unflatten(-2, (-1, BLOCK)) * scale[ids][..., None, None]).flatten(-3, -2)


def _decode(s):
    B, H, n_kv, page = s["case"]["batch"], s["H"], s["n_kv"], s["case"]["page"]
    width = s["page_table"].shape[1]
    mask = torch.arange(width * page, device=DEV)[None] < s["kv_lens"][:, None]      # [B, L]
    ids = s["page_table"].long().clamp_min(0)

    def cached(pages, scale):
        return _take(pages, scale, ids).transpose(1, 2).reshape(B, n_kv, width * page, D)

    q = s["q"].float().view(B, n_kv, H // n_kv, D)
    scores = torch.matmul(q, cached(s["k_pages"], s["k_scale"]).transpose(2, 3)) / math.sqrt(D)
    o = torch.matmul(_softmax(scores, mask[:, None, None]), cached(s["v_pages"], s["v_scale"]))
    return o.to(torch.bfloat16).view(B, H * D)


def _bounds(s):
    page, start = s["case"]["page"], s["start_pos"].long()
    n = torch.ones_like(start) if s["decode"] else s["cu_seqlens"].long().diff()
    j = torch.arange(s["page_table"].shape[1], device=DEV)[None]
    whole = (j >= (start // page)[:, None]) & (j < ((start + n) // page)[:, None])
    ids = s["page_table"].long()[whole]
    k = _take(s["k_pages"], s["k_scale"], ids)
    s["k_bounds"][ids, :, 0], s["k_bounds"][ids, :, 1] = k.amin(2).to(torch.bfloat16), k.amax(2).to(torch.bfloat16)
    return s["k_bounds"]


def _sparse(s):
    B, H, n_kv, page, select = s["case"]["batch"], s["H"], s["n_kv"], s["case"]["page"], s["case"]["select"]
    group, width = H // n_kv, s["page_table"].shape[1]
    lens = s["kv_lens"].long()
    pages = -(-lens // page)                                             # [B]
    table = s["page_table"].long().clamp_min(0)
    q = s["q"].view(B, n_kv, group, D)
    # (in 64 bits, rounded once: the places next to the last one selected lie close to each other)
    bounds = s["k_bounds"][table].double().transpose(1, 2)               # [B, n_kv, width, 2, 128]
    qd = q.double()
    score = torch.matmul(bounds[..., 1, :], qd.clamp_min(0).transpose(2, 3).contiguous()) + \
        torch.matmul(bounds[..., 0, :], qd.clamp_max(0).transpose(2, 3).contiguous())
    score = score.float().amax(-1)                                       # [B, n_kv, width]
    j = torch.arange(width, device=DEV)
    score = score.masked_fill((j >= pages[:, None])[:, None], float("-inf"))
    score = score.masked_fill((j == pages[:, None] - 1)[:, None], float("inf"))
    kept = torch.sort(score, dim=-1, descending=True, stable=True)[1][..., :select]
    kept = torch.sort(kept, dim=-1)[0]                                   # [B, n_kv, <= select]
    S = kept.shape[-1]
    ids = torch.gather(table[:, None].expand(B, n_kv, width), 2, kept)
    pos = kept[..., None] * page + torch.arange(page, device=DEV)
    mask = (pos < lens[:, None, None, None]).view(B, n_kv, S * page)
    head = torch.arange(n_kv, device=DEV)[None, :, None]

    def cached(pool, scale):
        codes = pool.dtype == torch.float8_e4m3fn
        held = (pool.view(torch.uint8)[ids, head].view(pool.dtype) if codes else pool[ids, head]).float()
        if scale is not None and scale.dim() == 1:
            held = held * scale[:, None, None, None]
        elif scale is not None:
            held = (held.unflatten(-2, (-1, BLOCK)) * scale[ids, head][..., None, None]).flatten(-3, -2)
        return held.view(B, n_kv, S * page, D)                           # (from [B, n_kv, S, page, 128])

    scores = torch.matmul(q.float(), cached(s["k_pages"], s["k_scale"]).transpose(2, 3)) / math.sqrt(D)
    o = torch.matmul(_softmax(scores, mask[:, :, None]), cached(s["v_pages"], s["v_scale"]))
    return o.to(torch.bfloat16).view(B, H * D)


# --- what a pass cannot do without ----------------------------------------------------------


def _held(case, positions):
    """Bytes of one head's keys, or values, of so many positions."""
    kind = case.get("cache", "block")
    return positions * D * (2 if kind == "bf16" else 1) + (4 * -(-positions // BLOCK) if kind == "block" else 0)


def work(case):
    lens, page = _lengths(case), case["page"]
    if case["kind"] == "assign":
        new, had = _roles(case), _starts(case)
        moved = sum(-(-a // page) if n < 0 else -(-(a + n) // page) - -(-a // page) for a, n in zip(had, new))
        tokens = len(new) if case["longest"] == 1 else sum(max(0, n) for n in new)
        return {"bytes": 8 * moved + 24 * len(new) + 8 * tokens, "flops": 0}
    H, n_kv = HEADS[case["model"]]
    T, row = sum(lens), 2 * D
    if case["kind"] == "decode":
        entries = sum(-(-n // page) for n in lens)
        return {"bytes": sum(2 * n_kv * _held(case, n) for n in lens) + 2 * len(lens) * H * row + 4 * (entries + len(lens)),
                "flops": 4 * T * H * D}
    if case["kind"] == "sparse":
        moved = flops = 0
        for n in lens:
            count = -(-n // page)
            seen = n if count <= case["select"] else (case["select"] - 1) * page + n - (count - 1) * page
            scored = 0 if count <= case["select"] else count - 1
            moved += 2 * n_kv * _held(case, seen) + scored * n_kv * 2 * row + 4 * count
            flops += 4 * seen * H * D + 4 * scored * H * D
        return {"bytes": moved + 2 * len(lens) * H * row + 4 * len(lens), "flops": flops}
    if case["kind"] == "bounds":
        whole = sum((a + n) // page - a // page for a, n in zip(_starts(case), lens))
        return {"bytes": whole * n_kv * (_held(case, page) + 2 * row) + 8 * len(lens), "flops": 2 * whole * n_kv * page * D}
    rows = 2 * n_kv * (row + D)                                          # k and v read, and stored
    if case["rotary"]:
        rows += 2 * H * row                                              # q read and written
        if case["longest"] > 1:
            rows += n_kv * row                                           # k written for the prompt's attention
    return {"bytes": T * rows + 2 * n_kv * 4 * sum(-(-n // BLOCK) for n in lens),
            "flops": T * (3 * (H + n_kv) * case["rotary"] + 2 * n_kv * D)}


# --- the definitions in 64 bits -------------------------------------------------------------


def _nearest_e4m3(x):
    """To the nearest of e4m3's values: 4 significant bits, steps of 2^-9 at least."""
    unit = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)
    return (torch.round(x / unit) * unit).clamp(-E4M3_MAX, E4M3_MAX)


def _exact_assign(case, s):
    page, table, free = case["page"], s["page_table"].tolist(), s["free_pages"].tolist()
    lens, new = s["lens"].tolist(), s["new_lens"].tolist()
    stack = free[:int(s["free_count"])]
    for b, n in enumerate(new):
        if n < 0 <= lens[b]:
            stack += table[b][:-(-lens[b] // page)]
    free[:len(stack)] = stack
    start, kv, after, slots, total, cu = [], [], [], [], 0, [0]
    room = len(stack)
    for b, n in enumerate(new):
        have = -(-lens[b] // page)
        need = -(-(lens[b] + max(0, n)) // page) - have
        room -= need
        ok = n > 0 and (need == 0 or room >= 0)
        if ok:
            for j in range(need):
                table[b][have + j] = stack.pop()
        start.append(lens[b] if ok else -1)
        kv.append(lens[b] + n if ok else 0)
        after.append(-1 if n < 0 else kv[-1] if ok else lens[b])
        rows = 1 if s["decode"] else max(0, n)
        slots += [table[b][(lens[b] + i) // page] * page + (lens[b] + i) % page if ok else -1 for i in range(rows)]
        total += rows
        cu.append(total)
    return {"start_pos": _ints(start), "kv_lens": _ints(kv), "cu_seqlens": None if s["decode"] else _ints(cu),
            "slots": torch.tensor(slots, dtype=torch.int64, device=DEV), "lens": _ints(after),
            "free_count": _ints([len(stack)]), "page_table": _ints(table), "free_pages": _ints(free)}


def _exact_append(case, s):
    T, n_kv, page, r = s["tokens"], s["n_kv"], case["page"], case["rotary"]
    lens, starts = _lengths(case), s["start_pos"].tolist()
    q, k, v = (s[x].double().view(T, -1, D) for x in ("q", "k", "v"))
    if r:
        at = torch.tensor([a + j for a, n in zip(starts, lens) for j in range(n)], dtype=torch.float64, device=DEV)
        first, second = (list(range(0, r, 2)), list(range(1, r, 2))) if case["interleaved"] else \
            (list(range(r // 2)), list(range(r // 2, r)))
        turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEV), at[:, None] * s["inv_freq"].double()).unsqueeze(1)
        for x in (q, k):
            z = torch.complex(x[..., first], x[..., second]) * turn
            x[..., first], x[..., second] = z.real, z.imag
    got = {"q": q.view(T, -1) if r else None, "k": k.view(T, -1) if r and case["longest"] > 1 else None}
    table = s["page_table"].tolist()
    for name, x in (("k", k), ("v", v)):
        pages, scales = s[name + "_pages"].double(), s[name + "_scale"].double()
        row = 0
        for b, (a, n) in enumerate(zip(starts, lens)):
            pos = a
            while pos < a + n:                                           # a block after another
                stop = min(a + n, pos // BLOCK * BLOCK + BLOCK)
                p, r0 = table[b][pos // page], pos % page // BLOCK * BLOCK
                new = x[row + pos - a:row + stop - a].transpose(0, 1)     # [n_kv, tokens, 128]
                size = new.abs().amax((1, 2)) / E4M3_MAX
                scale = torch.exp2(torch.ceil(torch.log2(size.clamp_min(LEAST))))
                if pos % BLOCK:
                    was = scales[p, :, r0 // BLOCK].clone()
                    scale = torch.maximum(scale, was)
                    old = pages[p, :, r0:r0 + pos % BLOCK]
                    pages[p, :, r0:r0 + pos % BLOCK] = _nearest_e4m3(old * (was / scale)[:, None, None])
                scales[p, :, r0 // BLOCK] = scale
                pages[p, :, pos % page:pos % page + stop - pos] = _nearest_e4m3(new / scale[:, None, None])
                pos = stop
            row += n
        got[name + "_pages"], got[name + "_scale"] = pages, scales
    return {n: got[n] for n in ("q", "k", "k_pages", "v_pages", "k_scale", "v_scale")}


def _exact_values(s, name, ids, heads=slice(None)):
    """Pages `ids` one after another, [heads, positions, 128]."""
    held = torch.stack([s[name + "_pages"][i, heads].to(torch.float32).double() for i in ids])
    scale = s[name + "_scale"]
    if scale is not None and scale.dim() == 1:
        held = held * scale[heads].double()[:, None, None]
    elif scale is not None:
        held = held * scale[ids][:, heads].double().repeat_interleave(BLOCK, dim=-1)[..., None]
    return held.transpose(0, 1).flatten(1, 2)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "assign":
        return _exact_assign(case, s)
    if case["kind"] == "append":
        return _exact_append(case, s)
    H, n_kv = HEADS[case["model"]]
    lens, page = _lengths(case), case["page"]
    table = s["page_table"].tolist()
    if case["kind"] == "bounds":
        got = s["k_bounds"].double()
        for b, (a, n) in enumerate(zip(s["start_pos"].tolist(), lens)):
            for j in range(a // page, (a + n) // page):
                k = _exact_values(s, "k", [table[b][j]])
                got[table[b][j], :, 0], got[table[b][j], :, 1] = k.min(1).values, k.max(1).values
        return got
    out = torch.zeros(case["batch"], n_kv, H // n_kv, D, dtype=torch.float64, device=DEV)
    q = s["q"].double().view(out.shape)
    for i, n in enumerate(lens):
        if not n:
            continue
        mine = table[i][:-(-n // page)]
        if case["kind"] == "decode" or len(mine) <= case["select"]:
            k, v = (_exact_values(s, x, mine)[:, :n] for x in ("k", "v"))
            w = torch.softmax(torch.bmm(q[i], k.transpose(1, 2).contiguous()) / D ** 0.5, dim=2)
            out[i] = torch.bmm(w, v)
            continue
        for g in range(n_kv):
            lo, hi = s["k_bounds"][mine[:-1], g].double().unbind(1)
            best = torch.stack([torch.where(x > 0, hi, lo) @ x for x in q[i, g]]).amax(0).float().tolist()
            kept = sorted(sorted(range(len(best)), key=lambda j: (-best[j], j))[:case["select"] - 1]) + [len(mine) - 1]
            ids = [mine[j] for j in kept]
            end = len(kept) * page - (len(mine) * page - n)
            k, v = (_exact_values(s, x, ids, slice(g, g + 1))[0, :end] for x in ("k", "v"))
            out[i, g] = torch.softmax(q[i, g] @ k.T / D ** 0.5, dim=1) @ v
    return out.view(case["batch"], H * D)
