"""Operators around an 8-bit key/value cache, as calls that can be timed and checked:

  tokens   one decoded token of each of several sequences: its key and value enter an 8-bit paged cache, its queries attend to the
           sequence (`cmlb200_attention_one` with cache_dtype CMLB200_DT_I8 or CMLB200_DT_E4M3)
  prompt   portions of prompts behind cached tokens: appended (`cmlb200_qk_norm_append`), then attended to (`cmlb200_attention_tiles`)
  fork     sequences branch: children share the parents' full pages and get their own copy of the page that is still being filled, in
           the pools of all layers (`cmlb200_pages_fork`)
  compact  pages of a fragmented cache move to the lowest free places, block tables follow (`cmlb200_pages_copy`)
  scores   log probabilities of given tokens, entropy and the best alternatives of rows of logits (`cmlb200_token_scores`)

The cache: pools [pages][page tokens][kv heads][head size] of 8-bit codes, scales [pages][page tokens / 16][kv heads] in fp32. A scale
is the smallest power of two whose multiples of up to 127 (int8) or 448 (e4m3) hold the 16 tokens' values of that head; where a later token
needs a larger one, the codes of the earlier ones are rounded to it."""
import math
import random

import torch

own = False

GROUP = 16                                                   # tokens that share a scale
FULL = {"i8": 127.0, "e4m3": 448.0}
LOGITS = {"f32": (torch.float32, 0), "bf16": (torch.bfloat16, 1), "f16": (torch.float16, 2)}

HEADS_32_8 = {"heads": 32, "kv_heads": 8, "dim": 128, "vdim": 128}
HEADS_16_4 = {"heads": 16, "kv_heads": 4, "dim": 128, "vdim": 128}


def listed():
    return [
        # One conversation's next token: latency.
        {"name": "tokens i8 b1 600", "kind": "tokens", "form": "i8", **HEADS_32_8, "page": 16, "batch": 1, "least": 600, "most": 600, "window": 0, "slopes": False, "sink": False},
        # A full batch behind long contexts: the bandwidth of the cache.
        {"name": "tokens i8 b32 8192", "kind": "tokens", "form": "i8", **HEADS_32_8, "page": 16, "batch": 32, "least": 8192, "most": 8192, "window": 0, "slopes": False, "sink": False},
        # A ragged batch of a model with windows, distance bias and sinks.
        {"name": "tokens e4m3 b23 ragged", "kind": "tokens", "form": "e4m3", **HEADS_16_4, "page": 64, "batch": 23, "least": 1, "most": 5000, "window": 1024, "slopes": True, "sink": True},
        # A new prompt.
        {"name": "prompt i8 512", "kind": "prompt", "form": "i8", **HEADS_32_8, "page": 16, "batch": 1, "least": 0, "most": 0, "rows": 512, "window": 0, "slopes": False, "sink": False},
        # Ragged portions behind cached tokens, small heads.
        {"name": "prompt e4m3 5x77 ragged", "kind": "prompt", "form": "e4m3", "heads": 12, "kv_heads": 4, "dim": 64, "vdim": 64, "page": 32, "batch": 5, "least": 5, "most": 1500, "rows": 77,
         "window": 0, "slopes": True, "sink": False},
        # A long prompt's second half.
        {"name": "prompt i8 4096 at 4096", "kind": "prompt", "form": "i8", **HEADS_32_8, "page": 16, "batch": 1, "least": 4096, "most": 4096, "rows": 4096, "window": 0, "slopes": False, "sink": False},
        # Four continuations of a prompt, every layer's pools.
        {"name": "fork 4 of 777", "kind": "fork", "layers": 32, "kv_heads": 8, "dim": 128, "page": 16, "parents": 1, "children": 4, "length": 777, "pages": 256},
        # A pool that long and short requests left in pieces.
        {"name": "compact 900", "kind": "compact", "layers": 16, "kv_heads": 8, "dim": 128, "page": 16, "pages": 2600, "moves": 900, "slots": 32},
        # The next token's candidates of one sequence: latency.
        {"name": "scores 1x32000 top5", "kind": "scores", "rows": 1, "vocab": 32000, "form": "f32", "top": 5},
        # One pass of the vocabulary projection over a prompt that is scored.
        {"name": "scores 256x32000 top20", "kind": "scores", "rows": 256, "vocab": 32000, "form": "f32", "top": 20},
        # An odd vocabulary, a decode batch.
        {"name": "scores 33x100003 top1", "kind": "scores", "rows": 33, "vocab": 100003, "form": "f32", "top": 1},
        # A long text scored, 16-bit logits.
        {"name": "scores 2000x128000 bf16", "kind": "scores", "rows": 2000, "vocab": 128000, "form": "bf16", "top": 0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["tokens"] * 4 + ["prompt"] * 3 + ["fork", "compact"] + ["scores"] * 3)
    if kind == "scores":
        rows, vocab = _log(rng, 1, 2000), _log(rng, 1000, 200000)
        if rng.random() < 0.5:
            vocab = vocab // 64 * 64
        form = rng.choice(["f32", "f32", "bf16", "f16"])
        while rows * vocab * (4 if form == "f32" else 2) > 500_000_000:
            rows = max(1, rows // 2)
        return {"kind": kind, "rows": rows, "vocab": vocab, "form": form, "top": rng.choice([0, 1, 5, 20, rng.randint(2, 32)])}
    if kind in ("fork", "compact"):
        c = {"kind": kind, "layers": rng.randint(2, 40), "kv_heads": rng.choice([1, 2, 4, 8]), "dim": rng.choice([64, 80, 128, 256]), "page": rng.choice([16, 32, 64])}
        page = 2 * c["layers"] * c["kv_heads"] * c["dim"] * c["page"]
        if kind == "fork":
            parents, children, length = rng.randint(1, 6), rng.randint(1, 8), _log(rng, 1, 1200)
            return {**c, "parents": parents, "children": children, "length": length, "pages": parents * (-(-length // c["page"])) + parents * children + 5}
        moves = max(1, min(_log(rng, 1, 900), 400_000_000 // page))
        return {**c, "moves": moves, "pages": 2 * moves + rng.randint(1, 300), "slots": rng.randint(1, 32)}
    group, kv_heads, dim = rng.choice([1, 2, 4, 4, 5, 8, 12]), rng.choice([1, 2, 4, 8]), rng.choice([64, 80, 128, 128, 128, 192, 256])
    c = {"kind": kind, "form": rng.choice(["i8", "e4m3"]), "heads": group * kv_heads, "kv_heads": kv_heads, "dim": dim, "vdim": dim if rng.random() < 0.8 else 64, "page": rng.choice([16, 16, 32, 64])}
    extra = {"window": rng.choice([0, 0, _log(rng, 16, 4096)]), "slopes": rng.random() < 0.3, "sink": rng.random() < 0.3}
    if kind == "tokens":
        most = _log(rng, 1, 20000)
        batch = max(1, min(_log(rng, 1, 64), 500_000_000 // (most * kv_heads * 2 * dim)))
        return {**c, "batch": batch, "least": rng.choice([most, rng.randint(1, most)]), "most": most, **extra}
    rows, most = _log(rng, 2, 3000), rng.choice([0, _log(rng, 1, 6000)])
    batch = rng.randint(1, 6)
    while batch * rows * (most + rows) * c["heads"] * dim > 4096 * 6000 * 32 * 128 or batch * rows * (most + rows) * c["heads"] > 6e8:
        batch, rows = max(1, batch // 2), max(2, rows // 2)
    return {**c, "batch": batch, "least": rng.choice([most, rng.randint(0, most)]), "most": most, "rows": rows, **extra}


# ---- what a user's program has in hand -------------------------------------------------------------------------------
def _pad16(n):
    return -(-n // 16) * 16


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _lengths(case, seed):
    """Cached tokens of every sequence in front of the call."""
    r = random.Random("%d lengths" % seed)
    got = [r.randint(case["least"], case["most"]) for _ in range(case["batch"])]
    got[0] = case["most"]
    return got


def prepare(case, seed):
    return {"tokens": _prepare_cache, "prompt": _prepare_cache, "fork": _prepare_fork, "compact": _prepare_compact, "scores": _prepare_scores}[case["kind"]](case, seed)


def _prepare_cache(case, seed):
    g, dev, page = _gen(seed), "cuda", case["page"]
    H, G, D, V = case["heads"], case["kv_heads"], case["dim"], case["vdim"]
    had, new = _lengths(case, seed), case.get("rows", 1)
    per = [-(-(n + new) // page) for n in had]               # pages of a sequence
    pages = sum(per) + 3
    order = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    table = torch.zeros(len(had), max(per), dtype=torch.int32, device=dev)
    at = 0
    for s, n in enumerate(per):
        table[s, :n] = order[at:at + n]
        at += n

    def pool(ld, width):
        codes = torch.randn(pages, page, G, ld, generator=g, device=dev)
        codes = codes.mul_(40).round_().clamp_(-127, 127).to(torch.int8) if case["form"] == "i8" else codes.mul_(130).clamp_(-448, 448).to(torch.float8_e4m3fn).view(torch.int8)
        codes[..., width:] = 0
        scale = torch.pow(2.0, torch.randint(-1, 2, (pages, page // GROUP, G), generator=g, device=dev).float()) * (2.0 ** -5 if case["form"] == "i8" else 2.0 ** -7)
        return codes, scale

    k_pool, k_scale = pool(_pad16(D), D)
    v_pool, v_scale = pool(_pad16(V), V)
    rows = torch.randn(len(had) * new, (H + G) * D + G * V, generator=g, device=dev)
    rows[:, :H * D] *= 1.5
    pos = torch.tensor([n + i for n in had for i in range(new)], dtype=torch.int32, device=dev)
    slot = torch.tensor([s for s in range(len(had)) for _ in range(new)], dtype=torch.int32, device=dev)
    tiles = torch.tensor([[s * new + k, min(64, new - k), s, n + k] for s, n in enumerate(had) for k in range(0, new, 64)], dtype=torch.int32, device=dev)
    # the 16-token groups that the call writes, with the tokens of each that were there before and that come
    touched = [(s, n, q) for s, n in enumerate(had) for q in range(n // GROUP, (n + new - 1) // GROUP + 1)]
    group = torch.tensor([(s, q) for s, _, q in touched], device=dev)
    group = table[group[:, 0], group[:, 1] * GROUP // page].long() * (page // GROUP) + group[:, 1] % (page // GROUP)
    token = torch.arange(GROUP, device=dev)[None] + torch.tensor([q * GROUP for _, _, q in touched], device=dev)[:, None]
    first = torch.tensor([n for _, n, _ in touched], device=dev)[:, None]
    base = torch.tensor([s * new - n for s, n, _ in touched], device=dev)[:, None]
    old, fresh = token < first, (token >= first) & (token < first + new)
    state = {"case": case, "k_pool": k_pool, "k_scale": k_scale, "v_pool": v_pool, "v_scale": v_scale, "rows": rows, "pos": pos, "slot": slot, "table": table, "tiles": tiles,
             "had": had, "new": new, "group": group, "old": old, "fresh": fresh, "row": torch.where(fresh, base + token, 0),
             "slopes": torch.pow(2.0, -8.0 * torch.arange(1, H + 1, device=dev).float() / H) if case["slopes"] else None,
             "out": torch.empty(len(had) * new, H * V, dtype=torch.bfloat16, device=dev)}
    return state


def _prepare_pools(case, seed):
    g, n = _gen(seed), 2 * case["layers"]
    bytes_ = case["page"] * case["kv_heads"] * case["dim"]
    codes = torch.randint(-127, 128, (n, case["pages"], bytes_), generator=g, device="cuda", dtype=torch.int8)
    scales = torch.rand(n, case["pages"], case["page"] // GROUP * case["kv_heads"], generator=g, device="cuda") + 0.5
    where = [(t[i].data_ptr(), t[i, 0].numel() * t.element_size(), t[i, 0].numel() * t.element_size()) for t in (codes, scales) for i in range(n)]
    return {"case": case, "codes": codes, "scales": scales, "pools": torch.tensor(where, dtype=torch.int64, device="cuda")}


def _prepare_fork(case, seed):
    state, r = _prepare_pools(case, seed), random.Random("%d pages" % seed)
    per, P, K = -(-case["length"] // case["page"]), case["parents"], case["children"]
    ids = r.sample(range(case["pages"]), P * per + P * K)
    table = torch.zeros(P * (K + 1), per + 2, dtype=torch.int32)
    table[:P, :per] = torch.tensor(ids[:P * per], dtype=torch.int32).view(P, per)
    full = case["length"] // case["page"]
    forks = [[p, P + p * K + k, full, ids[P * per + p * K + k] if full < per else -1] for p in range(P) for k in range(K)]
    state["forks"] = torch.tensor(forks, dtype=torch.int32).cuda()
    state["table"] = table.cuda()
    return state


def _prepare_compact(case, seed):
    """`moves` live pages in the upper part of the pool, as many free ones below them."""
    state, r = _prepare_pools(case, seed), random.Random("%d pages" % seed)
    n, pages = case["moves"], case["pages"]
    live = sorted(r.sample(range(pages - n), pages - 2 * n)) + list(range(pages - n, pages))   # n holes among the lower ones
    holes = sorted(set(range(pages - n)) - set(live))
    state["moves"] = torch.tensor([[a, b] for a, b in zip(range(pages - n, pages), holes)], dtype=torch.int32).cuda()
    r.shuffle(live)
    per = -(-len(live) // case["slots"])
    state["table"] = torch.tensor((live + live)[:per * case["slots"]], dtype=torch.int32).view(case["slots"], per).cuda()
    return state


def _prepare_scores(case, seed):
    g, (dtype, _) = _gen(seed), LOGITS[case["form"]]
    logits = torch.randn(case["rows"], case["vocab"], generator=g, device="cuda")
    logits = logits.mul_(2.5).add_(torch.randn(case["rows"], 1, generator=g, device="cuda") * 4).to(dtype)
    tokens = torch.randint(0, case["vocab"], (case["rows"],), generator=g, device="cuda", dtype=torch.int32)
    logits[torch.arange(case["rows"], device="cuda"), tokens.long()] += 6.0  # texts that are scored are likely ones
    logits[:, case["vocab"] // 2:case["vocab"] // 2 + 7] = -math.inf         # tokens that are not allowed
    logits[torch.arange(case["rows"], device="cuda"), tokens.long()] = logits[torch.arange(case["rows"], device="cuda"), tokens.long()].clamp_min(-20)
    new = lambda *shape, dtype=torch.float32: torch.empty(*shape, dtype=dtype, device="cuda")
    return {"case": case, "logits": logits, "tokens": tokens, "logprob": new(case["rows"]), "entropy": new(case["rows"]), "ids": new(case["rows"], case["top"], dtype=torch.int32),
            "best": new(case["rows"], case["top"])}


# ---- one pass ----------------------------------------------------------------------------------------------------------
def run(state):
    return {"tokens": _run_cache, "prompt": _run_cache, "fork": _run_fork, "compact": _run_compact, "scores": _run_scores}[state["case"]["kind"]](state)


def _package():
    import __graft_entry__ as entry
    return entry.load_package()


def _attn(state, pkg):
    """The layer's descriptor, which a program keeps."""
    if "attn" not in state:
        c = state["case"]
        state["attn"] = pkg.Attn(heads=c["heads"], kv_heads=c["kv_heads"], dim=c["dim"], vdim=c["vdim"], dim_ld=state["k_pool"].shape[-1], vdim_ld=state["v_pool"].shape[-1],
                                 scale=c["dim"] ** -0.5, window=c["window"], slopes=state["slopes"].data_ptr() if c["slopes"] else None, sink=int(c["sink"]), gate_col=-1,
                                 cache_dtype=pkg.DT_I8 if c["form"] == "i8" else pkg.DT_E4M3, k_pool=state["k_pool"].data_ptr(), v_pool=state["v_pool"].data_ptr(),
                                 k_scale=state["k_scale"].data_ptr(), v_scale=state["v_scale"].data_ptr(), block_size=c["page"], block_table=state["table"].data_ptr(),
                                 table_ld=state["table"].shape[1])
    return state["attn"]


def _run_cache(state):
    if own:
        pkg, stream = _package(), torch.cuda.current_stream().cuda_stream
        a, x, out, n = _attn(state, pkg), state["rows"], state["out"], state["rows"].shape[0]
        pos, slot = state["pos"].data_ptr(), state["slot"].data_ptr()
        if state["case"]["kind"] == "tokens":
            pkg.check(pkg.lib.cmlb200_attention_one(a, x.data_ptr(), x.stride(0), pos, slot, n, max(state["had"]), out.data_ptr(), out.stride(0), stream), "attention_one")
        else:
            pkg.check(pkg.lib.cmlb200_qk_norm_append(a, x.data_ptr(), x.stride(0), pos, slot, n, stream), "qk_norm_append")
            pkg.check(pkg.lib.cmlb200_attention_tiles(a, x.data_ptr(), x.stride(0), state["tiles"].data_ptr(), state["tiles"].shape[0], out.data_ptr(), out.stride(0), stream), "attention_tiles")
    else:
        _append(state)
        out = _attend(state)
    return {"out": out, "keys": _written(state, "k"), "values": _written(state, "v")}


def _values(codes, form):
    """What codes stand for, the scale aside."""
    return codes.float() if form == "i8" else codes.view(torch.float8_e4m3fn).float()


def _codes(x, form):
    return x.round().to(torch.int8) if form == "i8" else x.to(torch.float8_e4m3fn).view(torch.int8)


def _written(state, which):
    """The groups of tokens that the call wrote into, as the cache holds them now."""
    pool, scale = state[which + "_pool"], state[which + "_scale"]
    G, ld = pool.shape[2:]
    return _values(pool.view(-1, GROUP, G, ld).index_select(0, state["group"]), state["case"]["form"]) * scale.view(-1, 1, G, 1).index_select(0, state["group"])


def _scale_for(most, form):
    """The smallest power of two s with most <= FULL s, at least 2^-126."""
    m, x = torch.frexp(most)                                 # most = m 2^x, 1/2 <= m < 1
    fits, edge = (7, 127 / 128) if form == "i8" else (9, 448 / 512)
    return torch.ldexp(torch.ones_like(most), (x - fits + (m > edge)).clamp_min(-126))


def _append(state):
    c, group, old, fresh = state["case"], state["group"], state["old"], state["fresh"]
    H, G, form = c["heads"], c["kv_heads"], c["form"]
    at = H * c["dim"]
    for which, width in (("k", c["dim"]), ("v", c["vdim"])):
        pool, scale = state[which + "_pool"], state[which + "_scale"]
        codes, scales = pool.view(-1, GROUP, G, pool.shape[-1]), scale.view(-1, G)
        x = state["rows"][:, at:at + G * width].reshape(-1, G, width)[state["row"]].clamp(-65504, 65504)     # [groups, 16, G, width]
        at += G * width
        most = torch.where(fresh[:, :, None], x.abs().amax(-1), 0.0).amax(1)
        need, was = _scale_for(most, form), scales[group]
        had = old.any(1)[:, None]
        now = torch.where(had, torch.maximum(need, was), need)
        kept = codes[group]
        again = _codes(_values(kept, form) * torch.where(had, was / now, 1.0)[:, None, :, None], form)
        new = _codes(x / now[:, None, :, None], form)
        kept = torch.where(old[:, :, None, None], again, kept)
        kept[..., :width] = torch.where(fresh[:, :, None, None], new, kept[..., :width])
        kept[..., width:] = torch.where(fresh[:, :, None, None], 0, kept[..., width:])
        codes[group] = kept
        scales[group] = now


def _attend(state):
    c, new, S = state["case"], state["new"], len(state["had"])
    H, G, D, V, page = c["heads"], c["kv_heads"], c["dim"], c["vdim"], c["page"]
    keys = max(state["had"]) + new
    had = torch.tensor(state["had"], device="cuda")
    pages = state["table"][:, :-(-keys // page)].long()

    def cached(which, width):                                # [sequences, keys, G, width], zeros behind a sequence's end
        x = _values(state[which + "_pool"][pages], c["form"]).view(S, -1, GROUP, G, state[which + "_pool"].shape[-1])
        x = x * state[which + "_scale"][pages].view(S, -1, 1, G, 1)
        x = x.reshape(S, -1, G, x.shape[-1])[:, :keys, :, :width]
        return torch.where((torch.arange(keys, device="cuda")[None] < had[:, None] + new)[:, :, None, None], x, 0.0)

    q = state["rows"][:, :H * D].view(S, new, G, H // G, D).permute(0, 2, 3, 1, 4).reshape(S, G, H // G * new, D)
    score = torch.matmul(q, cached("k", D).permute(0, 2, 3, 1)).view(S, G, H // G, new, keys) * (D ** -0.5)
    i = had[:, None] + torch.arange(new, device="cuda")[None]                                              # positions
    back = i[:, :, None] - torch.arange(keys, device="cuda")[None, None]                                   # [S, new, keys]
    if c["slopes"]:
        score = score - state["slopes"].view(1, G, H // G, 1, 1) * back[:, None, None].float()
    seen = (back >= 0) & ((back < c["window"]) if c["window"] > 0 else True)
    score = torch.where(seen[:, None, None], score, -math.inf)
    most = score.amax(-1, keepdim=True)
    if c["sink"]:
        most = most.clamp_min(0.0)
    p = torch.exp(score - most)
    total = p.sum(-1, keepdim=True)
    if c["sink"]:
        total = total + torch.exp(-most)
    out = torch.matmul((p / total).view(S, G, H // G * new, keys), cached("v", V).permute(0, 2, 1, 3)).view(S, H, new, V)
    return out.permute(0, 2, 1, 3).reshape(S * new, H * V).to(torch.bfloat16)


def _pages(state, pkg):
    if "pages" not in state:
        t = state["table"]
        state["pages"] = pkg.Pages(pools=state["pools"].shape[0], pool=state["pools"].data_ptr(), most=state["codes"].shape[2], pages=state["case"]["pages"], table=t.data_ptr(), slots=t.shape[0],
                                   table_ld=t.shape[1])
    return state["pages"]


def _run_fork(state):
    forks, table = state["forks"], state["table"]
    if own:
        pkg = _package()
        pkg.check(pkg.lib.cmlb200_pages_fork(_pages(state, pkg), forks.data_ptr(), forks.shape[0], torch.cuda.current_stream().cuda_stream), "pages_fork")
    else:
        parent, child, shared, fresh = forks.long().unbind(1)
        place = torch.arange(table.shape[1], device="cuda")[None]
        rows = torch.where(place < shared[:, None], table[parent], table[child])
        copied = fresh >= 0
        rows = torch.where((place == shared[:, None]) & copied[:, None], fresh[:, None].int(), rows)
        if state["case"]["length"] % state["case"]["page"]:
            source = table[parent, shared].long()
            state["codes"][:, fresh] = state["codes"][:, source]
            state["scales"][:, fresh] = state["scales"][:, source]
        table[child] = rows
    return {"codes": state["codes"], "scales": state["scales"], "table": table}


def _run_compact(state):
    moves, table = state["moves"], state["table"]
    if own:
        pkg = _package()
        pkg.check(pkg.lib.cmlb200_pages_copy(_pages(state, pkg), moves.data_ptr(), moves.shape[0], torch.cuda.current_stream().cuda_stream), "pages_copy")
    else:
        a, b = moves.long().unbind(1)
        state["codes"][:, b] = state["codes"][:, a]
        state["scales"][:, b] = state["scales"][:, a]
        name = torch.arange(state["case"]["pages"], dtype=torch.int32, device="cuda")
        name[a] = moves[:, 1]
        table.copy_(name[table.long()])
    return {"codes": state["codes"], "scales": state["scales"], "table": table}


def _run_scores(state):
    c, x, tokens = state["case"], state["logits"], state["tokens"]
    if own:
        pkg = _package()
        pkg.check(pkg.lib.cmlb200_token_scores(x.data_ptr(), LOGITS[c["form"]][1], x.stride(0), c["rows"], c["vocab"], tokens.data_ptr(), c["top"], state["logprob"].data_ptr(),
                                               state["entropy"].data_ptr(), state["ids"].data_ptr(), state["best"].data_ptr(), torch.cuda.current_stream().cuda_stream), "token_scores")
        got = {"logprob": state["logprob"], "entropy": state["entropy"]}
        return {**got, "ids": state["ids"], "best": state["best"]} if c["top"] else got
    x = x.float()
    d = x - x.amax(-1, keepdim=True)
    e = torch.exp(d)
    total = e.sum(-1, keepdim=True)
    lp = d - torch.log(total)
    got = {"logprob": lp.gather(1, tokens.long()[:, None])[:, 0], "entropy": torch.log(total[:, 0]) - torch.where(e > 0, e * d, 0.0).sum(-1) / total[:, 0]}
    if c["top"]:
        values, ids = torch.sort(lp, dim=-1, descending=True, stable=True)
        got.update(ids=ids[:, :c["top"]].int(), best=values[:, :c["top"]].clone())
    return got


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    if kind == "scores":
        return {"bytes": case["rows"] * (case["vocab"] * (4 if case["form"] == "f32" else 2) + 12 + 8 * case["top"]), "flops": 6 * case["rows"] * case["vocab"]}
    if kind in ("fork", "compact"):
        page = 2 * case["layers"] * (case["page"] * case["kv_heads"] * case["dim"] + case["page"] // GROUP * case["kv_heads"] * 4)
        if kind == "compact":
            return {"bytes": 2 * case["moves"] * page + 8 * (case["pages"] - case["moves"]), "flops": 0}
        n = case["parents"] * case["children"] if case["length"] % case["page"] else 0
        full = case["length"] // case["page"]                # a source page that several children copy is read once
        return {"bytes": (n + (case["parents"] if n else 0)) * page + 4 * full * case["parents"] * (1 + case["children"]) + 16, "flops": 0}
    H, G, D, V, new, w = case["heads"], case["kv_heads"], case["dim"], case["vdim"], case.get("rows", 1), case["window"]
    # lengths are those of a middling seed: what they are drawn between
    had = [case["most"]] + [(case["least"] + case["most"]) // 2] * (case["batch"] - 1)
    pairs = sum(min(n + i + 1, w) if w > 0 else n + i + 1 for n in had for i in range(new))
    keys = sum(min(n + new, w + new - 1) if w > 0 else n + new for n in had)
    return {"bytes": keys * G * (D + V + 8 / GROUP) + case["batch"] * new * (4 * ((H + G) * D + G * V) + 2 * H * V), "flops": 2 * pairs * H * (D + V)}


# ---- from the definition, in 64 bits ---------------------------------------------------------------------------------------
def exact(case, seed):
    if case["kind"] in ("fork", "compact"):
        return None
    state = prepare(case, seed)
    return _exact_scores(case, state) if case["kind"] == "scores" else _exact_cache(case, state)


def _exact_scores(case, state):
    lp, entropy = [], []
    best = []
    for r0 in range(0, case["rows"], 256):
        x = state["logits"][r0:r0 + 256].double()
        z = torch.logsumexp(x, -1)
        p = torch.exp(x - z[:, None])
        lp.append(x[torch.arange(len(x)), state["tokens"][r0:r0 + 256].long()] - z)
        entropy.append(-torch.special.xlogy(p, p).sum(-1))
        best.append(torch.topk(x, case["top"], -1).values - z[:, None] if case["top"] else None)
    got = {"logprob": torch.cat(lp), "entropy": torch.cat(entropy)}
    return {**got, "ids": None, "best": torch.cat(best)} if case["top"] else got


def _exact_cache(case, state):
    H, G, D, V, page, new = case["heads"], case["kv_heads"], case["dim"], case["vdim"], case["page"], state["new"]
    top, tiny = FULL[case["form"]], 2.0 ** -126
    outs, written = [], {"k": [], "v": []}
    x = state["rows"].double()
    for s, n in enumerate(state["had"]):
        mine, seq = x[s * new:(s + 1) * new], {}
        ids = state["table"][s, :-(-(n + new) // page)].long()
        for which, width, at in (("k", D, H * D), ("v", V, (H + G) * D)):
            ld = state[which + "_pool"].shape[-1]
            raw = state[which + "_pool"][ids].view(-1, G, ld)
            raw = (raw if case["form"] == "i8" else raw.view(torch.float8_e4m3fn)).double()
            unit = state[which + "_scale"][ids].view(-1, G).double()                                        # per group
            q0, q1 = n // GROUP, (n + new - 1) // GROUP + 1
            fresh = torch.zeros(q1 * GROUP - q0 * GROUP, G, ld, dtype=torch.float64, device="cuda")
            fresh[n - q0 * GROUP:n - q0 * GROUP + new, :, :width] = mine[:, at:at + G * width].view(new, G, width).clamp(-65504, 65504)
            most = fresh.view(-1, GROUP, G, ld).abs().amax((1, 3))
            need = torch.exp2(torch.ceil(torch.log2(torch.clamp(most / top, min=tiny))))
            need = torch.where(need / 2 * top >= most, need / 2, need).clamp_min(tiny)                        # log2 may round up at a border
            need = torch.where(need * top < most, need * 2, need)
            was = unit[q0:q1].clone()
            now = need.clone()
            if n % GROUP:
                now[0] = torch.maximum(need[0], was[0])
                ratio = (was[0] / now[0])[None, :, None]
                part = raw[q0 * GROUP:n] * ratio
                raw[q0 * GROUP:n] = part.round() if case["form"] == "i8" else part.float().to(torch.float8_e4m3fn).double()
            code = fresh[n - q0 * GROUP:n - q0 * GROUP + new] / now.repeat_interleave(GROUP, 0)[n - q0 * GROUP:n - q0 * GROUP + new, :, None]
            raw[n:n + new] = code.round() if case["form"] == "i8" else code.float().to(torch.float8_e4m3fn).double()
            unit[q0:q1] = now
            held = raw * unit.repeat_interleave(GROUP, 0)[:, :, None]
            written[which].append(held[q0 * GROUP:q1 * GROUP].view(-1, GROUP, G, ld))
            seq[which] = held[:n + new, :, :width]
        o = torch.empty(new, H, V, dtype=torch.float64, device="cuda")
        for r0 in range(0, new, 512):
            i = torch.arange(n + r0, n + min(r0 + 512, new), device="cuda")
            gap = i[:, None] - torch.arange(n + new, device="cuda")[None]
            hidden = (gap < 0) | ((gap >= case["window"]) if case["window"] > 0 else (gap < 0))
            for h in range(H):
                z = mine[r0:r0 + 512, h * D:(h + 1) * D] @ seq["k"][:, h // (H // G)].T / math.sqrt(D)
                if case["slopes"]:
                    z -= float(state["slopes"][h]) * gap
                z = z.masked_fill(hidden, -math.inf)
                if case["sink"]:
                    z = torch.cat([z, torch.zeros(len(z), 1, dtype=torch.float64, device="cuda")], 1)
                o[r0:r0 + 512, h] = torch.softmax(z, -1)[:, :n + new] @ seq["v"][:, h // (H // G)]
        outs.append(o.reshape(new, H * V))
    return {"out": torch.cat(outs), "keys": torch.cat(written["k"]), "values": torch.cat(written["v"])}
