"""Operators of a model in 8-bit integers and of drafted tokens, as calls that can be timed and checked:

  linear   y = x W^T with int8 codes on both sides: rows of x (tokens) are quantised in the call, rows of W (channels) when the model was
           loaded, each with a scale of its own (`cmlb200_linear_dense8`); with a bias and a cap where the weight has them
  glu      the same for a feed-forward's gate and up rows: bf16 act(gate) * up (`cmlb200_linear_dense8_glu`)
  verify   drafted tokens of several sequences against the target's logits: how many are kept, and the token behind them
           (`cmlb200_verify_drafts`); a sequence without drafts has a token drawn

Codes: scale = a / 127 and code = round(127 v / a), ties to even, a = the largest magnitude of the row, at least 127 * 2^-126.

Verification: p and q are the softmax of target's and drafter's logits over the temperature (q is 1 at the draft where drafts come without
logits). Draft i is kept while u_i q(draft) < p(draft). What follows the kept ones is drawn from p where all were kept, otherwise from what
p has above q, as the token with the largest weight / E, E = -log(1 - v) being standard exponentials. A sequence brings one 64-bit random
number, the key of Philox4x32-10: v of token j is word j mod 4 of counter (j / 4, 0, 0, 0), u_i word i mod 4 of counter (i / 4, 1, 0, 0);
v = (word + 1/2) / 2^32, u = word / 2^32. A temperature of 0 keeps drafts while they are the largest logit's token, and takes that."""
import math
import random

import numpy as np
import torch

own = False

TYPES = {"f32": (torch.float32, 0), "bf16": (torch.bfloat16, 1), "f16": (torch.float16, 2)}
ACTS = {"silu": 0, "gelu": 1}
TINY = 127 * 2.0 ** -126


def listed():
    return [
        # One token through a square projection of a 7B model: latency.
        {"name": "linear m1 4096x4096", "kind": "linear", "m": 1, "rows": 4096, "cols": 4096, "form": "bf16", "bias": False, "cap": 0.0},
        # A decode batch through its down projection.
        {"name": "linear m8 4096x11008", "kind": "linear", "m": 8, "rows": 4096, "cols": 11008, "form": "bf16", "bias": False, "cap": 0.0},
        # A step of drafted tokens through a vocabulary projection with bias and cap, odd sizes, 16-bit floats.
        {"name": "linear m29 10007x1501 f16", "kind": "linear", "m": 29, "rows": 10007, "cols": 1501, "form": "f16", "bias": True, "cap": 30.0},
        # A short prompt.
        {"name": "linear m77 11008x4096", "kind": "linear", "m": 77, "rows": 11008, "cols": 4096, "form": "bf16", "bias": False, "cap": 0.0},
        # A prompt through query, key and value rows of a model with biases.
        {"name": "linear m500 6144x4096 bias", "kind": "linear", "m": 500, "rows": 6144, "cols": 4096, "form": "bf16", "bias": True, "cap": 0.0},
        # A long prompt through a 70B model's down projection.
        {"name": "linear m4096 8192x28672", "kind": "linear", "m": 4096, "rows": 8192, "cols": 28672, "form": "bf16", "bias": False, "cap": 0.0},
        # One token through a 7B model's gate and up projections.
        {"name": "glu m1 11008x4096", "kind": "glu", "m": 1, "ff": 11008, "cols": 4096, "form": "bf16", "act": "silu"},
        # A ragged batch of prompts through a small feed-forward of odd sizes.
        {"name": "glu m333 1003x777 gelu", "kind": "glu", "m": 333, "ff": 1003, "cols": 777, "form": "bf16", "act": "gelu"},
        # A prompt through a 7B model's gate and up projections.
        {"name": "glu m2048 11008x4096", "kind": "glu", "m": 2048, "ff": 11008, "cols": 4096, "form": "bf16", "act": "silu"},
        # One conversation, four drafts with the drafter's logits: latency.
        {"name": "verify b1 4 drafts 32000", "kind": "verify", "sequences": 1, "least": 4, "most": 4, "vocab": 32000, "form": "f32", "drafter": True, "greedy": 0.0},
        # A full batch with a large vocabulary.
        {"name": "verify b32 4 drafts 128000", "kind": "verify", "sequences": 32, "least": 4, "most": 4, "vocab": 128000, "form": "f32", "drafter": True, "greedy": 0.0},
        # A ragged batch, drafts that a lookup proposed, some sequences greedy, an odd vocabulary, 16-bit logits.
        {"name": "verify b23 0 to 7 drafts 100003 bf16", "kind": "verify", "sequences": 23, "least": 0, "most": 7, "vocab": 100003, "form": "bf16", "drafter": False, "greedy": 0.25},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "glu", "verify"])
    if kind == "verify":
        c = {"kind": kind, "sequences": _log(rng, 1, 64), "most": rng.choice([0, 1, 3, 4, 5, 8, rng.randint(1, 12)]), "vocab": _log(rng, 1000, 160000), "form": rng.choice(["f32", "f32", "bf16", "f16"]),
             "drafter": rng.random() < 0.6, "greedy": rng.choice([0.0, 0.0, 0.3, 1.0])}
        c["least"] = rng.choice([c["most"], rng.randint(0, c["most"])])
        while c["sequences"] * (c["most"] + 1) * c["vocab"] > 20_000_000:
            c["sequences"] = max(1, c["sequences"] // 2)
            c["vocab"] = c["vocab"] if c["sequences"] > 1 else c["vocab"] // 2
        return c
    m, rows, cols = rng.choice([_log(rng, 1, 32), _log(rng, 1, 4096)]), _log(rng, 48, 32000), _log(rng, 48, 30000)
    if rng.random() < 0.5:
        rows, cols = max(1, rows // 64) * 64, max(1, cols // 64) * 64
    while rows * cols > 230_000_000 or m * rows * cols > 4096 * 8192 * 28672:
        rows, cols = rows // 2 + 1, cols // 2 + 1
    if kind == "glu":
        return {"kind": kind, "m": m, "ff": rows // 2, "cols": cols, "form": rng.choice(["bf16", "bf16", "f16"]), "act": rng.choice(["silu", "gelu"])}
    return {"kind": kind, "m": m, "rows": rows, "cols": cols, "form": rng.choice(["bf16", "bf16", "f16"]), "bias": rng.random() < 0.3, "cap": rng.choice([0.0, 0.0, 0.0, 30.0])}


# ---- what a user's program has in hand -------------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def prepare(case, seed):
    return _prepare_verify(case, seed) if case["kind"] == "verify" else _prepare_linear(case, seed)


def _prepare_linear(case, seed):
    g, m, cols = _gen(seed), case["m"], case["cols"]
    glu = case["kind"] == "glu"
    half = -(-case["ff"] // 16) * 16 if glu else 0           # gate and up rows in turns of 16
    rows = 2 * half if glu else case["rows"]
    ld = -(-cols // 128) * 128
    codes = torch.zeros(-(-rows // 16) * 16, ld, dtype=torch.int8, device="cuda")
    scale = torch.zeros(codes.shape[0], device="cuda")
    for r0 in range(0, rows, 4096):                          # (the model's loader did this once)
        w = torch.randn(min(4096, rows - r0), cols, generator=g, device="cuda") * 0.02
        a = w.abs().amax(1).clamp_min(TINY)
        codes[r0:r0 + len(w), :cols] = torch.round(w * 127 / a[:, None]).to(torch.int8)
        scale[r0:r0 + len(w)] = a / 127
    if glu and half != case["ff"]:                           # groups that are not full end in rows of zeros
        turns, s = codes.view(-1, 2, 16, ld), scale.view(-1, 2, 16)
        turns[-1, :, case["ff"] % 16:] = 0
        s[-1, :, case["ff"] % 16:] = 2.0 ** -126
    x = torch.randn(m, cols, generator=g, device="cuda")
    x[:, torch.randint(0, cols, (max(1, cols // 500),), generator=g, device="cuda")] *= 6.0       # the channels that stand out
    state = {"case": case, "codes": codes, "scale": scale, "n": rows, "x": x.to(TYPES[case["form"]][0]),
             "bias": torch.randn(rows, generator=g, device="cuda") if case.get("bias") else None,
             "y": torch.empty(m, case["ff"], dtype=torch.bfloat16, device="cuda") if glu else torch.empty(m, rows, device="cuda")}
    return state


def _counts(case, seed):
    r = random.Random("%d drafts" % seed)
    n = [r.randint(case["least"], case["most"]) for _ in range(case["sequences"])]
    n[0] = case["most"]
    return n


def _prepare_verify(case, seed):
    g, V, counts = _gen(seed), case["vocab"], _counts(case, seed)
    S, rows, drafts = len(counts), sum(counts) + len(counts), sum(counts)
    r = random.Random("%d temperatures" % seed)
    temperature = [0.0 if r.random() < case["greedy"] else r.choice([0.7, 1.0, 1.0, 1.3]) for _ in range(S)]
    first = [0]
    for n in counts:
        first.append(first[-1] + n + 1)
    target_row = torch.tensor([first[s] + i for s, n in enumerate(counts) for i in range(n)], dtype=torch.long, device="cuda")
    heat = torch.tensor([temperature[s] for s, n in enumerate(counts) for _ in range(n)], device="cuda")
    kind = TYPES[case["form"]][0]
    logits = torch.empty(rows, V, dtype=kind, device="cuda")
    for r0 in range(0, rows, 64):                            # a few likely tokens above a broad field
        part = torch.randn(min(64, rows - r0), V, generator=g, device="cuda")
        logits[r0:r0 + 64] = (2.0 * part + 0.35 * part.pow(3)).to(kind)
    draft_logits = torch.empty(max(drafts, 1), V, dtype=kind, device="cuda")
    tokens = torch.zeros(max(drafts, 1), dtype=torch.int32, device="cuda")
    for r0 in range(0, drafts, 64):
        at = target_row[r0:r0 + 64]
        d = (logits[at].float() + 0.5 * torch.randn(len(at), V, generator=g, device="cuda")).to(kind)
        draft_logits[r0:r0 + 64] = d
        noise = -torch.log(torch.empty(len(at), V, device="cuda").exponential_(generator=g))
        tokens[r0:r0 + 64] = torch.argmax(d.float() + heat[r0:r0 + 64, None] * noise, 1).int()        # what a drafter with these logits drew
    state = {"case": case, "counts": counts, "first": torch.tensor(first, dtype=torch.int32, device="cuda"), "logits": logits, "tokens": tokens,
             "draft_logits": draft_logits if case["drafter"] else None, "temperature": torch.tensor(temperature, device="cuda"),
             "random": torch.randint(-2 ** 63, 2 ** 63 - 1, (S,), generator=g, device="cuda", dtype=torch.int64),
             "accepted": torch.empty(S, dtype=torch.int32, device="cuda"), "next": torch.empty(S, dtype=torch.int32, device="cuda")}
    # where the plain form finds things: a sequence's places among rows and drafts
    state["row_of"] = torch.tensor([s for s, n in enumerate(counts) for _ in range(n + 1)], device="cuda")
    state["draft_of"] = torch.tensor([s for s, n in enumerate(counts) for _ in range(n)], dtype=torch.long, device="cuda")
    state["place_of"] = torch.tensor([i for n in counts for i in range(n)], dtype=torch.long, device="cuda")
    state["target_row"] = target_row
    return state


# ---- one pass -----------------------------------------------------------------------------------------------------------
def _package():
    import __graft_entry__
    return __graft_entry__.load_package()


def run(state):
    if own:
        return _own_verify(state) if state["case"]["kind"] == "verify" else _own_linear(state)
    return _plain_verify(state) if state["case"]["kind"] == "verify" else _plain_linear(state)


def _own_linear(state):
    pkg, c, x, y = _package(), state["case"], state["x"], state["y"]
    if "weight" not in state:                                # the handle that a program keeps, and room for the rows' codes
        state["weight"] = pkg.Dense8(rows=state["n"], cols=c["cols"], ld=state["codes"].shape[1], w=state["codes"].data_ptr(), scale=state["scale"].data_ptr(),
                                     bias=state["bias"].data_ptr() if state["bias"] is not None else None, cap=c.get("cap", 0.0))
        state["work"] = torch.empty(pkg.lib.cmlb200_dense8_work_bytes(c["m"], state["n"], c["cols"]), dtype=torch.uint8, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    if c["kind"] == "glu":
        pkg.check(pkg.lib.cmlb200_linear_dense8_glu(state["weight"], x.data_ptr(), TYPES[c["form"]][1], x.stride(0), c["m"], c["ff"], ACTS[c["act"]], y.data_ptr(), y.stride(0),
                                                    state["work"].data_ptr(), stream), "linear_dense8_glu")
    else:
        pkg.check(pkg.lib.cmlb200_linear_dense8(state["weight"], x.data_ptr(), TYPES[c["form"]][1], x.stride(0), c["m"], y.data_ptr(), y.stride(0), state["work"].data_ptr(), stream), "linear_dense8")
    return y


def _plain_linear(state):
    c = state["case"]
    x = state["x"].float()
    a = x.abs().amax(1, keepdim=True).clamp_min(TINY)
    code, unit = torch.round(x * 127 / a), a / 127
    w, s = state["codes"][:, :c["cols"]], state["scale"]
    if c["kind"] == "linear":
        y = torch.matmul(code, w[:c["rows"]].float().T) * (unit * s[:c["rows"]])
        if state["bias"] is not None:
            y = y + state["bias"]
        return c["cap"] * torch.tanh(y / c["cap"]) if c["cap"] else y
    w, s = w.reshape(-1, 2, 16, c["cols"]), s.view(-1, 2, 16)
    gate, up = (torch.matmul(code, w[:, i].reshape(-1, c["cols"])[:c["ff"]].float().T) * (unit * s[:, i].reshape(-1)[:c["ff"]]) for i in (0, 1))
    if c["act"] == "gelu":
        act = 0.5 * gate * (1 + torch.tanh(math.sqrt(2 / math.pi) * (gate + 0.044715 * gate.pow(3))))
    else:
        act = gate / (1 + torch.exp(-gate))
    return (act * up).to(torch.bfloat16)


def _own_verify(state):
    pkg, c, x, d = _package(), state["case"], state["logits"], state["draft_logits"]
    if "drafts" not in state:
        state["drafts"] = pkg.Drafts(sequences=c["sequences"], rows=x.shape[0], first=state["first"].data_ptr(), tokens=state["tokens"].data_ptr(), logits=d.data_ptr() if d is not None else None,
                                     ld=d.stride(0) if d is not None else 0, temperature=state["temperature"].data_ptr(), random=state["random"].data_ptr())
        state["work"] = torch.empty(pkg.lib.cmlb200_verify_work_bytes(x.shape[0], c["sequences"]), dtype=torch.uint8, device="cuda")
    pkg.check(pkg.lib.cmlb200_verify_drafts(state["drafts"], x.data_ptr(), TYPES[c["form"]][1], x.stride(0), c["vocab"], state["accepted"].data_ptr(), state["next"].data_ptr(),
                                            state["work"].data_ptr(), torch.cuda.current_stream().cuda_stream), "verify_drafts")
    return {"accepted": state["accepted"], "next": state["next"]}


def _philox(key, c0, c1):
    """The four words of Philox4x32-10 at counters (c0, c1, 0, 0); 64-bit keys, everything in int64."""
    low = 0xFFFFFFFF
    k0, k1 = key & low, (key >> 32) & low
    c = [c0, torch.zeros_like(c0) + c1, torch.zeros_like(c0), torch.zeros_like(c0)]
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [((b >> 32) & low) ^ c[1] ^ k0, b & low, ((a >> 32) & low) ^ c[3] ^ k1, a & low]
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack(torch.broadcast_tensors(*c), -1)


def _plain_verify(state):
    c, V, S, dev = state["case"], state["case"]["vocab"], state["case"]["sequences"], "cuda"
    heat, key, first = state["temperature"].double(), state["random"], state["first"].long()
    greedy, row_of, draft_of, place_of, at = heat <= 0, state["row_of"], state["draft_of"], state["place_of"], state["target_row"]
    most = max(state["counts"])
    place = torch.arange(V, device=dev)

    def lowest_best(v):
        return torch.where(v == v.amax(-1, keepdim=True), place, V).amin(-1)

    def softmax(x, t):
        z = x.double() / torch.where(t > 0, t, 1.0)[:, None]
        e = torch.exp(z - z.amax(-1, keepdim=True))
        return e / e.sum(-1, keepdim=True)

    best = lowest_best(state["logits"])
    accepted = torch.zeros(S, dtype=torch.long, device=dev)
    if most:
        n = len(at)
        token = state["tokens"][:n].long()
        p = torch.cat([softmax(state["logits"][at[i:i + 32]], heat[draft_of[i:i + 32]]).gather(1, token[i:i + 32, None]) for i in range(0, n, 32)])[:, 0]
        q = torch.ones_like(p)
        if c["drafter"]:
            q = torch.cat([softmax(state["draft_logits"][i:i + 32], heat[draft_of[i:i + 32]]).gather(1, token[i:i + 32, None]) for i in range(0, n, 32)])[:, 0]
        word = _philox(key[draft_of], place_of // 4, 1).gather(1, (place_of % 4)[:, None])[:, 0]
        kept = torch.where(greedy[draft_of], best[at] == token, word.double() * 2.0 ** -32 * q < p)
        grid = torch.zeros(S, most, dtype=torch.long, device=dev)
        grid[draft_of, place_of] = kept.long()
        accepted = torch.cumprod(grid, 1).sum(1)
    stop = first[:-1] + accepted
    short = stop + 1 < first[1:]                             # a draft was turned down
    weight = softmax(state["logits"][stop], heat)
    if most:
        turned = torch.where(short, stop - torch.arange(S, device=dev), 0)
        if c["drafter"]:
            less = (weight - softmax(state["draft_logits"][turned], heat)).clamp_min(0.0)
        else:
            less = torch.where(place[None] == state["tokens"][turned].long()[:, None], 0.0, weight)
        less = torch.where(less.amax(1, keepdim=True) > 0, less, weight)
        weight = torch.where(short[:, None], less, weight)
    v = _philox(key[:, None], torch.arange(-(-V // 4), device=dev)[None], 0).reshape(S, -1)[:, :V]
    drawn = lowest_best(weight / -torch.log1p(-(v.double() + 0.5) * 2.0 ** -32))
    return {"accepted": accepted.int(), "next": torch.where(greedy, best[stop], drawn).int()}


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------
def work(case):
    if case["kind"] == "verify":
        # counts are those of a middling seed: what they are drawn between
        drafts = case["most"] + (case["sequences"] - 1) * (case["least"] + case["most"]) // 2
        values = (drafts * (2 if case["drafter"] else 1) + case["sequences"]) * case["vocab"]
        return {"bytes": values * (4 if case["form"] == "f32" else 2) + 4 * drafts + 24 * case["sequences"], "flops": 4 * values}
    m, cols = case["m"], case["cols"]
    rows = 2 * case["ff"] if case["kind"] == "glu" else case["rows"]
    out = 2 * case["ff"] if case["kind"] == "glu" else 4 * rows
    return {"bytes": rows * (cols + 4) + 2 * m * cols + m * out + (4 * rows if case.get("bias") else 0), "flops": 2 * m * rows * cols}


# ---- from the definition, in 64 bits ---------------------------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    return _exact_verify(case, state) if case["kind"] == "verify" else _exact_linear(case, state)


def _exact_linear(case, state):
    x, outs = state["x"].double(), []
    most = torch.clamp(x.abs().max(1).values, min=TINY)
    held = torch.round(x * (127.0 / 1) / most[:, None])      # a 16-bit number times 127 over a 16-bit number: ties are exact
    step = (state["n"] + 7) // 8 // 32 * 32 + 32
    for r0 in range(0, state["n"], step):
        w = state["codes"][r0:r0 + step, :case["cols"]].double()[:state["n"] - r0]
        outs.append((held @ w.T) * state["scale"][r0:r0 + len(w)].double() * (most / 127)[:, None])
    y = torch.cat(outs, 1)
    if case["kind"] == "linear":
        if state["bias"] is not None:
            y += state["bias"].double()
        return torch.tanh(y / case["cap"]) * case["cap"] if case["cap"] else y
    y = y.view(len(y), -1, 2, 16)
    g, u = y[:, :, 0].reshape(len(y), -1)[:, :case["ff"]], y[:, :, 1].reshape(len(y), -1)[:, :case["ff"]]
    s = torch.sigmoid(2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)) if case["act"] == "gelu" else torch.sigmoid(g)
    return g * s * u


def _exact_verify(case, state):
    """Sequence by sequence on the host, random numbers with unsigned words."""
    def words(key, c0, c1):
        c = [c0.astype(np.uint64), np.full_like(c0, c1, dtype=np.uint64), np.zeros(len(c0), np.uint64), np.zeros(len(c0), np.uint64)]
        mask, k = np.uint64(2 ** 32 - 1), [key % 2 ** 32, key >> 32]
        for _ in range(10):
            a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
            c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & mask, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), a & mask]
            k = [(k[0] + 0x9E3779B9) % 2 ** 32, (k[1] + 0xBB67AE85) % 2 ** 32]
        return np.stack(c, 1).reshape(-1)

    V, first = case["vocab"], state["first"].tolist()
    accepted, following = [], []
    for s, n in enumerate(state["counts"]):
        x = state["logits"][first[s]:first[s + 1]].double().cpu().numpy()
        d = state["draft_logits"][first[s] - s:first[s] - s + n].double().cpu().numpy() if case["drafter"] else None
        drafts = state["tokens"][first[s] - s:first[s] - s + n].tolist()
        t, key = float(state["temperature"][s]), int(state["random"][s]) % 2 ** 64
        if t <= 0:
            i = 0
            while i < n and int(np.argmax(x[i])) == drafts[i]:
                i += 1
            accepted.append(i)
            following.append(int(np.argmax(x[i])))
            continue

        def chances(row):
            e = np.exp((row - row.max()) / t)
            return e / e.sum()

        u = words(key, np.arange(-(-n // 4)), 1) / 2.0 ** 32 if n else []
        i, q = 0, None
        p = chances(x[0])
        while i < n:
            q = chances(d[i]) if case["drafter"] else np.eye(1, V, drafts[i])[0]
            if not u[i] * q[drafts[i]] < p[drafts[i]]:
                break
            i += 1
            p, q = chances(x[i]), None
        w = p if q is None else np.maximum(p - q, 0) if case["drafter"] else np.where(q > 0, 0, p)
        w = w if w.max() > 0 else p
        e = -np.log1p(-(words(key, np.arange(-(-V // 4)), 0)[:V] + 0.5) / 2.0 ** 32)
        accepted.append(i)
        following.append(int(np.argmax(w / e)))
    return {"accepted": torch.tensor(accepted, dtype=torch.int32), "next": torch.tensor(following, dtype=torch.int32)}
