"""Performance cases of the batched-serving attention operators: a paged KV cache, the attention of new
tokens over it, and the attention over packed prompts.

Kinds:

  append   keys and values of new tokens stored in a paged KV cache, with the position rotation of q
           and k on the way: one token per sequence (decode), or packed prompts
  decode   attention of one new token per sequence over its pages, each sequence its own length
  prefill  causal attention over packed prompts of different lengths

Head counts are those of perf/cases.py's models (40 / 8, 16 / 4 and 32 / 8 heads of 128).  Activations
and cached keys and values are N(0, 1); e4m3 caches hold them under a scale per KV head.  Pages are
scattered over the pool as after some time of serving.
"""
import math

import torch

own = False

DEV = "cuda:0"
D = 128
E4M3_MAX = 448.0
HEADS = {"h3136": (40, 8), "h2048": (16, 4), "h2560": (32, 8)}


def listed():
    return [
        # one interactive conversation's next token, rotated, far into a long context: the smallest call
        {"name": "append_1_token", "kind": "append", "model": "h3136", "cache": "bf16", "page": 16, "batch": 1,
         "shortest": 1, "longest": 1, "start": 100000, "rotary": 128, "interleaved": False},
        # a decode step of a serving batch on an 8-bit cache, partial rotation of neighbouring pairs
        {"name": "append_48_tokens_e4m3", "kind": "append", "model": "h2560", "cache": "e4m3", "page": 32, "batch": 48,
         "shortest": 1, "longest": 1, "start": 30000, "rotary": 64, "interleaved": True},
        # a batch of prompts of a model without rotation: keys and values only
        {"name": "append_5_prompts", "kind": "append", "model": "h3136", "cache": "bf16", "page": 64, "batch": 5,
         "shortest": 61, "longest": 1801, "start": 0, "rotary": 0, "interleaved": False},
        # one long document into an 8-bit cache, its rotated q and k returned for the attention over it
        {"name": "append_long_prompt_e4m3", "kind": "append", "model": "h3136", "cache": "e4m3", "page": 128, "batch": 1,
         "shortest": 8191, "longest": 8191, "start": 0, "rotary": 128, "interleaved": False},
        # one conversation of some hundred tokens: a call that latency bounds
        {"name": "decode_1x777", "kind": "decode", "model": "h3136", "cache": "bf16", "page": 16, "batch": 1,
         "shortest": 777, "longest": 777, "idle": 0},
        # a small batch of chats, in a step captured for more sequences than are active
        {"name": "decode_16_chats", "kind": "decode", "model": "h2048", "cache": "bf16", "page": 64, "batch": 16,
         "shortest": 150, "longest": 2900, "idle": 3},
        # a large serving batch on an 8-bit cache
        {"name": "decode_64_e4m3", "kind": "decode", "model": "h3136", "cache": "e4m3", "page": 32, "batch": 64,
         "shortest": 90, "longest": 8000, "idle": 0},
        # long documents beside a new conversation: one sequence holds most of the positions
        {"name": "decode_long", "kind": "decode", "model": "h3136", "cache": "bf16", "page": 128, "batch": 3,
         "shortest": 17, "longest": 60001, "idle": 0},
        # a few short turns at once: launch and latency
        {"name": "prefill_4_turns", "kind": "prefill", "model": "h2048", "batch": 4, "shortest": 5, "longest": 77},
        # chat prompts of a serving step
        {"name": "prefill_12_prompts", "kind": "prefill", "model": "h3136", "batch": 12, "shortest": 33, "longest": 700},
        # retrieval prompts, ragged
        {"name": "prefill_4_long", "kind": "prefill", "model": "h2560", "batch": 4, "shortest": 300, "longest": 2500},
        # two documents: the quadratic part is everything
        {"name": "prefill_2_documents", "kind": "prefill", "model": "h3136", "batch": 2, "shortest": 5000, "longest": 8200},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "decode", "prefill"])
    case = {"kind": kind, "model": rng.choice(["h3136", "h2048", "h2560"])}
    if kind == "prefill":
        case["batch"] = _log(rng, 1, 32)
        case["longest"] = _log(rng, 1, 8192 // max(2, case["batch"]))
        case["shortest"] = rng.randint(1, case["longest"])
        return case
    case["cache"] = rng.choice(["bf16", "e4m3"])
    case["page"] = rng.choice([16, 32, 64, 128, 256])
    case["batch"] = _log(rng, 1, 64)
    if kind == "append":
        prompts = rng.random() < 0.5
        case["longest"] = _log(rng, 2, 8192 // case["batch"]) if prompts else 1
        case["shortest"] = rng.randint(1, case["longest"])
        case["start"] = rng.choice([0, _log(rng, 1, 120000)]) if prompts else _log(rng, 1, 120000)
        case["rotary"] = rng.choice([0, 32, 64, 96, 128, 128])
        case["interleaved"] = rng.random() < 0.5
    else:
        case["longest"] = _log(rng, 1, min(60000, 120000 // case["batch"]))
        case["shortest"] = _log(rng, 1, case["longest"]) if case["longest"] > 1 else 1
        case["idle"] = rng.choice([0, 0, rng.randint(0, case["batch"] - 1)])
    return case


def _lengths(case):
    """The sequences' lengths, from the longest to the shortest over their logarithm, in scattered order."""
    n, lo, hi = case["batch"], case["shortest"], case["longest"]
    step = next(s for s in (7, 5, 3, 1) if math.gcd(s, n) == 1)
    lens = [int(round(hi * (lo / hi) ** ((step * i % n) / max(1, n - 1)))) for i in range(n)]
    for i in range(case.get("idle", 0)):
        lens[n - 1 - i] = 0
    return lens


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


def _scales(gen, n_kv):
    """Scales per KV head that spread N(0, 1) values over e4m3's range."""
    return 0.01 + 0.02 * torch.rand(n_kv, generator=gen, device=DEV)


def _pool(case, gen, n_pages, n_kv):
    """K and V pages [n_pages, n_kv, page, 128] that hold earlier tokens, and their scales (None: bf16)."""
    pages = [_normal(gen, n_pages, n_kv, case["page"], D) for _ in range(2)]
    if case["cache"] == "bf16":
        return [p.to(torch.bfloat16) for p in pages], [None, None]
    scales = [_scales(gen, n_kv) for _ in range(2)]
    return [(p / s[:, None, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn) for p, s in zip(pages, scales)], scales


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    H, n_kv = HEADS[case["model"]]
    lens = _lengths(case)
    state = {"case": dict(case), "H": H, "n_kv": n_kv}
    if case["kind"] == "decode":
        counts = [-(-n // case["page"]) for n in lens]
        (state["k_pages"], state["v_pages"]), (state["k_scale"], state["v_scale"]) = _pool(case, gen, max(1, sum(counts)), n_kv)
        # every sequence's pages, scattered over the pool; the entries after its last page are not in use
        order = torch.randperm(max(1, sum(counts)), generator=gen, device=DEV).to(torch.int32)
        width = max(1, max(counts))
        used = torch.arange(width, device=DEV)[None] < _ints(counts)[:, None]
        state["page_table"] = torch.full((case["batch"], width), -1, dtype=torch.int32, device=DEV)
        state["page_table"][used] = order[:sum(counts)]
        state["kv_lens"] = _ints(lens)
        state["q"] = _normal(gen, case["batch"], H * D).to(torch.bfloat16)
        return state
    T = sum(lens)
    qkv = _normal(gen, T, (H + 2 * n_kv) * D).to(torch.bfloat16)       # as one projection writes them
    state["q"], state["k"], state["v"] = qkv[:, :H * D], qkv[:, H * D:(H + n_kv) * D], qkv[:, (H + n_kv) * D:]
    state["cu_seqlens"] = _ints(_cumulative(lens))
    if case["kind"] == "prefill":
        return state
    page = case["page"]
    # start positions around case["start"], no two alike; the pages of the new tokens are each sequence's own
    starts = [0 if not case["start"] else case["start"] + 37 * i for i in range(case["batch"])]
    spans = [(s // page, -(-(s + n) // page)) for s, n in zip(starts, lens)]
    n_pages = sum(b - a for a, b in spans) + 3
    (state["k_pages"], state["v_pages"]), (state["k_scale"], state["v_scale"]) = _pool(case, gen, n_pages, n_kv)
    order = torch.randperm(n_pages, generator=gen, device=DEV).to(torch.int32)
    state["page_table"] = torch.full((case["batch"], max(b for _, b in spans)), int(order[-1]), dtype=torch.int32, device=DEV)
    at = 0
    for i, (a, b) in enumerate(spans):
        state["page_table"][i, a:b] = order[at:at + b - a]
        at += b - a
    state["start_pos"] = _ints(starts)
    state["decode"] = case["longest"] == 1
    state["inv_freq"] = None
    if case["rotary"]:
        state["inv_freq"] = 10000.0 ** (-torch.arange(0, case["rotary"], 2, device=DEV, dtype=torch.float32) / case["rotary"])
    return state


# --- one pass -------------------------------------------------------------------------------


def run(state):
    if own:
        return _run_own(state)
    return {"append": _append, "decode": _decode, "prefill": _prefill}[state["case"]["kind"]](state)


def _run_own(state):
    from nemotron_infer_amd import ops

    s = state
    kind = s["case"]["kind"]
    if kind == "prefill":
        return ops.sdpa_prefill_packed_bf16(s["q"], s["k"], s["v"], s["cu_seqlens"], s["H"], s["n_kv"])
    if kind == "decode":
        return ops.sdpa_decode_paged(s["q"], s["k_pages"], s["v_pages"], s["page_table"], s["kv_lens"],
                                     k_scale=s["k_scale"], v_scale=s["v_scale"])
    rotate = s["inv_freq"] is not None
    # a decode step needs no k of its own afterwards: the attention reads the cache
    k_out = torch.empty(s["k"].shape, dtype=torch.bfloat16, device=DEV) if rotate and not s["decode"] else None
    q_out, k_out = ops.kv_append_paged(s["k"], s["v"], s["k_pages"], s["v_pages"], s["page_table"], s["start_pos"],
                                       cu_seqlens=None if s["decode"] else s["cu_seqlens"],
                                       q=s["q"] if rotate else None, inv_freq=s["inv_freq"],
                                       interleaved=s["case"]["interleaved"], k_scale=s["k_scale"], v_scale=s["v_scale"],
                                       k_out=k_out)
    return {"q": q_out, "k": k_out, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _tokens(cu_seqlens, T):
    """Sequence and place in it of every packed token."""
    t = torch.arange(T, device=DEV)
    b = torch.searchsorted(cu_seqlens[1:].long(), t, right=True)
    return b, t - cu_seqlens.long()[b]


def _rotate(x, cos, sin, interleaved):
    """x [T, heads, 128] float32; cos, sin [T, 1, rotary / 2]."""
    half = cos.shape[-1]
    turned = x[..., :2 * half]
    a, b = (turned[..., 0::2], turned[..., 1::2]) if interleaved else (turned[..., :half], turned[..., half:])
    pair = (a * cos - b * sin, a * sin + b * cos)
    turned = torch.stack(pair, dim=-1).flatten(-2) if interleaved else torch.cat(pair, dim=-1)
    return torch.cat((turned, x[..., 2 * half:]), dim=-1)


def _append(s):
    case, T = s["case"], s["k"].shape[0]
    b, place = _tokens(s["cu_seqlens"], T)
    pos = s["start_pos"].long()[b] + place
    k, v = (s[n].float().view(T, s["n_kv"], D) for n in ("k", "v"))
    q_out = k_out = None
    if s["inv_freq"] is not None:
        angle = pos.double()[:, None] * s["inv_freq"].double()
        cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
        q_out = _rotate(s["q"].float().view(T, s["H"], D), cos, sin, case["interleaved"]).to(torch.bfloat16).view(T, -1)
        k = _rotate(k, cos, sin, case["interleaved"])
        if not s["decode"]:
            k_out = k.to(torch.bfloat16).view(T, -1)
    page = s["page_table"].long()[b, pos // case["page"]]
    for pages, scale, x in ((s["k_pages"], s["k_scale"], k), (s["v_pages"], s["v_scale"], v)):
        if scale is None:
            pages[page, :, pos % case["page"]] = x.to(torch.bfloat16)
        else:
            codes = (x / scale[:, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
            pages.view(torch.uint8)[page, :, pos % case["page"]] = codes.view(torch.uint8)
    return {"q": q_out, "k": k_out, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _softmax(scores, mask):
    """Weights of the last axis where mask is true; a row without any gets zeros."""
    scores = scores.masked_fill(~mask, float("-inf"))
    top = scores.amax(dim=-1, keepdim=True).clamp_min(torch.finfo(scores.dtype).min)
    weights = (scores - top).exp()
    return weights / weights.sum(dim=-1, keepdim=True).clamp_min(torch.finfo(scores.dtype).tiny)


def _decode(s):
    case, H, n_kv = s["case"], s["H"], s["n_kv"]
    B, page = case["batch"], case["page"]
    at = torch.arange(s["page_table"].shape[1] * page, device=DEV)
    mask = at[None] < s["kv_lens"][:, None]                              # [B, L]
    ids = s["page_table"].long().clamp_min(0)[:, at // page]

    def cached(pages, scale):
        x = pages.view(torch.uint8)[ids, :, at % page].view(pages.dtype) if scale is not None else pages[ids, :, at % page]
        x = x.float().permute(0, 2, 1, 3)                                # [B, n_kv, L, 128]
        return x * scale[:, None, None] if scale is not None else x

    q = s["q"].float().view(B, n_kv, H // n_kv, D)
    scores = torch.matmul(q, cached(s["k_pages"], s["k_scale"]).transpose(2, 3)) / math.sqrt(D)
    o = torch.matmul(_softmax(scores, mask[:, None, None]), cached(s["v_pages"], s["v_scale"]))
    return o.to(torch.bfloat16).view(B, H * D)


def _prefill(s):
    H, n_kv, T = s["H"], s["n_kv"], s["q"].shape[0]
    B, L = s["case"]["batch"], s["case"]["longest"]
    b, place = _tokens(s["cu_seqlens"], T)

    def padded(x, heads):
        out = torch.zeros(B, L, heads, D, device=DEV)
        out[b, place] = x.float().view(T, heads, D)
        return out.permute(0, 2, 1, 3)

    q = padded(s["q"], H).reshape(B, n_kv, H // n_kv * L, D)
    scores = torch.matmul(q, padded(s["k"], n_kv).transpose(2, 3)).view(B, H, L, L) / math.sqrt(D)
    at = torch.arange(L, device=DEV)
    weights = _softmax(scores, (at[None] <= at[:, None])[None, None])
    o = torch.matmul(weights.view(B, n_kv, H // n_kv * L, L), padded(s["v"], n_kv)).view(B, H, L, D)
    return o[b, :, place].to(torch.bfloat16).view(T, H * D)


# --- what a pass cannot do without ----------------------------------------------------------


def work(case):
    H, n_kv = HEADS[case["model"]]
    lens = _lengths(case)
    T = sum(lens)
    row = 2 * D
    if case["kind"] == "prefill":
        pairs = sum(n * (n + 1) // 2 for n in lens)
        return {"bytes": T * (2 * H + 2 * n_kv) * row + 4 * (len(lens) + 1), "flops": 4 * H * D * pairs}
    held = D * (2 if case["cache"] == "bf16" else 1)
    if case["kind"] == "decode":
        entries = sum(-(-n // case["page"]) for n in lens)
        return {"bytes": 2 * T * n_kv * held + 2 * len(lens) * H * row + 4 * (entries + len(lens)),
                "flops": 4 * T * H * D}
    rows = 2 * n_kv * (row + held)                                       # k and v read, and stored
    if case["rotary"]:
        rows += 2 * H * row                                              # q read and written
        if case["longest"] > 1:
            rows += n_kv * row                                           # k written for the prompt's attention
    return {"bytes": T * rows, "flops": T * 3 * (H + n_kv) * case["rotary"]}


# --- the definitions in 64 bits -------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    H, n_kv = HEADS[case["model"]]
    lens = _lengths(case)
    if case["kind"] == "prefill":
        out = torch.empty(sum(lens), H, D, dtype=torch.float64, device=DEV)
        first = 0
        for n in lens:
            q, k, v = (s[x][first:first + n].double().view(n, -1, D) for x in ("q", "k", "v"))
            later = torch.ones(n, n, dtype=torch.bool, device=DEV).triu(1)
            for h in range(H):
                e = q[:, h] @ k[:, h * n_kv // H].T * D ** -0.5
                e[later] = -math.inf
                out[first:first + n, h] = torch.softmax(e, dim=1) @ v[:, h * n_kv // H]
            first += n
        return out.view(-1, H * D)
    if case["kind"] == "decode":
        out = torch.zeros(case["batch"], H, D, dtype=torch.float64, device=DEV)
        for i, n in enumerate(lens):
            if not n:
                continue
            mine = s["page_table"][i, :-(-n // case["page"])].tolist()
            held = []
            for pages, scale in ((s["k_pages"], s["k_scale"]), (s["v_pages"], s["v_scale"])):
                rows = torch.cat([pages[p] for p in mine], dim=1) if scale is None else \
                    torch.cat([pages[p].to(torch.float32) for p in mine], dim=1)
                rows = rows[:, :n].double()
                held.append(rows if scale is None else rows * scale.double().view(-1, 1, 1))
            q = s["q"][i].double().view(n_kv, H // n_kv, D)
            w = torch.softmax(torch.bmm(q, held[0].transpose(1, 2).contiguous()) / D ** 0.5, dim=2)
            out[i] = torch.bmm(w, held[1]).view(H, D)
        return out.view(case["batch"], H * D)
    T = sum(lens)
    starts = s["start_pos"].tolist()
    where = torch.tensor([(i, starts[i] + j) for i, n in enumerate(lens) for j in range(n)], device=DEV)
    r = case["rotary"]
    q, k, v = (s[x].double().view(T, -1, D) for x in ("q", "k", "v"))
    if r:
        first, second = (list(range(0, r, 2)), list(range(1, r, 2))) if case["interleaved"] else \
            (list(range(r // 2)), list(range(r // 2, r)))
        turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEV),
                           where[:, 1:].double() * s["inv_freq"].double()).unsqueeze(1)
        for x in (q, k):
            z = torch.complex(x[..., first], x[..., second]) * turn
            x[..., first], x[..., second] = z.real, z.imag
    got = {"q": q.view(T, -1) if r else None, "k": k.view(T, -1) if r and case["longest"] > 1 else None}
    for name, x, scale in (("k_pages", k, s["k_scale"]), ("v_pages", v, s["v_scale"])):
        pages = s[name].double()
        if scale is not None:                   # to the nearest of e4m3's values: 4 significant bits, steps of 2^-9 at least
            x = (x / scale.double()[:, None]).clamp(-E4M3_MAX, E4M3_MAX)
            unit = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)
            x = torch.round(x / unit) * unit
        ids = s["page_table"][where[:, 0], where[:, 1] // case["page"]].long()
        pages[ids, :, where[:, 1] % case["page"]] = x
        got[name] = pages
    return got
