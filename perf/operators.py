"""The paged KV cache in 8 bits, as cases that can be timed and compared: keys
and values quantised as they are appended and read back, attention of single
tokens and drafts over the quantised pages, and attention of chunks of new
tokens over them.

A cached head vector is stored as 8-bit floats (e4m3: 4 exponent bits, 3
mantissa bits, largest value 448) with one power-of-two scale: for the vector x
of one token and KV head, e is the least integer with max|x| <= 448 * 2^e (at
least -126), and element d is stored as round(x[d] / 2^e) to the nearest e4m3
value, ties to even.  The stored value is code * 2^e.

A case is a dict of plain values.  ``listed()`` names the fixed ones,
``draw(rng)`` gives more of the same ranges, ``prepare(case, seed)`` makes what
a program holds before the call, ``run(state)`` is one pass, through the
public entry points where ``own`` is true and in plain torch where it is not,
``exact(case, seed)`` the same results in 64 bits, and ``work(case)`` the bytes
and operations that a pass cannot do without.
"""

import math
import random

import torch

own = False

# The model shapes of this repository's benchmark and tests (query heads, KV
# heads, head_dim), and generic ones: one KV head for 20 query heads, a
# head_dim that is no multiple of 64, an odd number of heads.
MODELS = {
    "qwen2-0.5b": (14, 2, 64),
    "llama3-8b": (32, 8, 128),
    "qwen3-8b": (32, 8, 128),
    "gemma2-9b": (16, 8, 256),
    "qwen2.5-32b": (40, 8, 128),
    "one kv head": (20, 1, 128),
    "head_dim 96": (12, 4, 96),
    "three heads": (9, 3, 80),
}
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def _case(name, kind, model, **kw):
    """`batch` sequences with contexts spread log-uniformly over [ctx_lo,
    ctx_hi] that each have `rows` new tokens, and `chunks` prefill chunks of
    `chunk` tokens after `prefix` cached ones.  kind "store": the new tokens
    are appended and read back; "attn": they attend, themselves included, over
    the filled cache; "step": they are appended and attend in one call, and are
    read back."""
    case = {"name": name, "kind": kind, "model": model, "page": 16, "x": "f16", "y": "f16", "batch": 0, "ctx_lo": 0,
            "ctx_hi": 0, "rows": 1, "chunks": 0, "chunk": 0, "prefix": 0, "window": 0, "softcap": 0.0}
    case.update(kw)
    return case


def listed():
    return [
        # One user's chat: one token appended to one layer.  Latency is all there is.
        _case("append one token", "store", "llama3-8b", batch=1, ctx_lo=2500, ctx_hi=2500, x="f32", y="f32"),
        # A serving batch's append on a small model.
        _case("append a batch", "store", "qwen2-0.5b", batch=64, ctx_lo=100, ctx_hi=4000, page=32),
        # A prompt's keys and values, and their way back out (a preempted sequence, 16-bit floats hold the
        # values exactly).
        _case("append a prompt", "store", "llama3-8b", chunks=1, chunk=4096, x="bf16", y="bf16"),
        # A few short conversations on a small model, append and attention in one call.
        _case("small batch step", "step", "qwen2-0.5b", batch=4, ctx_lo=128, ctx_hi=512, x="f32", y="f32"),
        # One sequence alone: few workgroups, a long axis.
        _case("one sequence decode", "attn", "llama3-8b", batch=1, ctx_lo=2500, ctx_hi=2500, page=32, x="f32", y="f32"),
        # A full decode batch.
        _case("full batch decode", "attn", "llama3-8b", batch=32, ctx_lo=4096, ctx_hi=4096),
        # Speculative decoding: four drafts a sequence, verified at once, soft-capped logits, head_dim 256.
        _case("draft verify", "attn", "gemma2-9b", batch=16, ctx_lo=8192, ctx_hi=8192, rows=4, softcap=50.0),
        # Documents: contexts of 131060 tokens.
        _case("long context decode", "attn", "qwen2.5-32b", batch=4, ctx_lo=131060, ctx_hi=131060, x="bf16", y="bf16"),
        # Ragged decode rows beside fresh chunks of 512 tokens, append included: a step of continuous batching.
        _case("continuous batch", "step", "qwen3-8b", batch=64, ctx_lo=256, ctx_hi=16384, chunks=8, chunk=512,
              x="bf16", y="bf16"),
        # A prompt from its first token, alone.
        _case("prompt prefill", "attn", "llama3-8b", chunks=1, chunk=4096),
        # A ragged chunk after a cached prefix, sliding window and soft-cap, f32 in and out.
        _case("chunk after prefix", "attn", "gemma2-9b", chunks=1, chunk=777, prefix=3001, window=4096, softcap=50.0,
              x="f32", y="f32"),
        # A short follow-up question after a long cached document, on an odd shape.
        _case("short chunk, long prefix", "attn", "head_dim 96", chunks=1, chunk=61, prefix=20011, page=64),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["store", "store", "decode", "decode", "verify", "step", "mixed", "prefill", "prefill"])
    model = rng.choice(sorted(MODELS))
    case = _case("", "attn", model, page=rng.choice([16, 16, 32, 64]), x=rng.choice(["f32", "f16", "bf16"]),
                 y=rng.choice(["f32", "f16", "bf16"]))
    del case["name"]
    if model == "gemma2-9b":
        case.update(softcap=50.0, window=rng.choice([0, 4096]))
    elif rng.random() < 0.2:
        case.update(window=_log_int(rng, 5, 3000))
    if kind == "store":
        case.update(kind="store", window=0, softcap=0.0)
        if rng.random() < 0.5:
            lo = _log_int(rng, 1, 4000)
            case.update(batch=_log_int(rng, 1, 200), ctx_lo=lo, ctx_hi=2 * lo, rows=rng.choice([1, 1, 1, 3, 4]))
        else:
            case.update(chunks=rng.choice([1, 1, 3]), chunk=_log_int(rng, 2, 4000), prefix=rng.choice([0, 7, 1001]))
        return case
    if kind in ("decode", "verify", "step", "mixed"):
        case["batch"] = _log_int(rng, 1, 64)
        longest = min(65536, 120000 // case["batch"])
        lo = _log_int(rng, 8, longest)
        case.update(ctx_lo=lo, ctx_hi=rng.randint(lo, min(longest, 8 * lo)))
    if kind == "verify":
        case["rows"] = rng.randint(2, 5)
    if kind == "step":
        case["kind"] = "step"
    if kind == "mixed":
        case.update(kind=rng.choice(["attn", "step"]), chunks=rng.randint(1, 4), chunk=_log_int(rng, 30, 600))
    if kind == "prefill":
        case.update(chunks=rng.choice([1, 1, 2, 4]), chunk=_log_int(rng, 20, 2000),
                    prefix=rng.choice([0, 0, _log_int(rng, 16, 6000)]))
    return case


# ------------------------------------------------------------------- inputs


def _rng_of(case):
    """Sizes within a case's ranges follow from the case alone."""
    return random.Random("/".join(f"{k}={case[k]}" for k in sorted(case) if k != "name"))


def _gen(seed, *more):
    g = torch.Generator(device="cuda")
    g.manual_seed(hash((int(seed),) + tuple(int(x) for x in more)) & 0x7FFFFFFFFFFF)
    return g


def _sequences(case):
    """(cached tokens, new tokens) of each sequence, decode rows first."""
    rng, lo, hi = _rng_of(case), case["ctx_lo"], case["ctx_hi"]
    seqs = [(min(hi, max(lo, _log_int(rng, max(lo, 1), max(hi, 1)))), case["rows"]) for _ in range(case["batch"])]
    return seqs + [(case["prefix"], case["chunk"])] * case["chunks"]


def _rows(case):
    """Position and sequence of every new row."""
    seqs = _sequences(case)
    return [c + i for c, n in seqs for i in range(n)], [s for s, (_, n) in enumerate(seqs) for _ in range(n)]


def _kv(g, n, nkv, hd, dt):
    """Keys and values of n tokens, [n, kv_heads, head_dim].  A key's channels
    differ (a few carry several times the others' magnitude), tokens differ in
    magnitude too, and an occasional value vector is all zeros."""
    chan = torch.exp2(torch.randn(nkv, hd, device="cuda", generator=g) * 0.7)
    k = torch.randn(n, nkv, hd, device="cuda", generator=g) * chan * 0.6
    v = torch.randn(n, nkv, hd, device="cuda", generator=g)
    v *= torch.exp2(torch.randn(n, nkv, 1, device="cuda", generator=g) * 0.5)
    v *= (torch.rand(n, nkv, 1, device="cuda", generator=g) > 0.002)
    return k.to(dt), v.to(dt)


def _cached(case, seed, s, n):
    _, nkv, hd = MODELS[case["model"]]
    return _kv(_gen(seed, 1, s), n, nkv, hd, DTYPES[case["x"]])


def _new(case, seed, m):
    """Queries, new keys and new values of a call's m rows."""
    nq, nkv, hd = MODELS[case["model"]]
    g, dt = _gen(seed, 2), DTYPES[case["x"]]
    q = (torch.randn(m, nq, hd, device="cuda", generator=g) * 1.2).to(dt)
    k, v = _kv(g, m, nkv, hd, dt)
    return q, k, v


def _pages(case):
    """The pages of every sequence: a busy engine's pool hands them out in no order."""
    page = case["page"]
    need = [-(-(c + n) // page) for c, n in _sequences(case)]
    ids = list(range(sum(need)))
    _rng_of(case).shuffle(ids)
    out = []
    for n in need:
        out.append(ids[:n])
        ids = ids[n:]
    return out


def prepare(case, seed):
    return _prepare_own(case, seed) if own else _prepare_plain(case, seed)


def _fill_lens(case):
    """Tokens of each sequence in the cache before a pass: "attn" finds its new tokens there already."""
    return [c + (n if case["kind"] == "attn" else 0) for c, n in _sequences(case)]


def _outputs(case, m):
    nq, nkv, hd = MODELS[case["model"]]
    dt = DTYPES[case["y"]]
    y = torch.zeros(m, nq, hd, dtype=dt, device="cuda")
    return y, torch.zeros(m, nkv, hd, dtype=dt, device="cuda"), torch.zeros(m, nkv, hd, dtype=dt, device="cuda")


def _contents(case, seed, k_new, v_new):
    """(sequence, first position, keys, values) of what the cache holds before a pass."""
    at = 0
    for s, (c, n) in enumerate(_sequences(case)):
        if case["kind"] != "store" and c:
            yield (s, 0) + _cached(case, seed, s, c)
        if case["kind"] == "attn":
            yield s, c, k_new[at:at + n], v_new[at:at + n]
        at += n


def _prepare_own(case, seed):
    from flint_amd import ops
    from flint_amd.pool import ArenaSpec, KvPool, RowMeta

    nq, nkv, hd = MODELS[case["model"]]
    seqs, page = _sequences(case), case["page"]
    total = [c + n for c, n in seqs]
    pages = sum(-(-n // page) for n in total)
    pool = KvPool(ArenaSpec(total, pages), nkv, hd, page_len=page, kv_dtype="e4m3")
    # pieces of the sequences allocated in random order
    piece = max(page, -(-max(sum(total), 1) // 4096 // page) * page)
    order = [s for s, n in enumerate(total) for _ in range(-(-n // piece))]
    _rng_of(case).shuffle(order)
    have = [0] * len(total)
    for s in order:
        n = min(piece, total[s] - have[s])
        pool.alloc(s, have[s], n)
        have[s] += n
    positions, owners = _rows(case)
    m = len(owners)
    q, k, v = _new(case, seed, m)
    fill = RowMeta(max(total))
    for s, t0, kc, vc in _contents(case, seed, k, v):
        n = kc.shape[0]
        fill.write(list(range(t0, t0 + n)), [s] * n)
        ops.kv_store(kc, vc, pool, 0, n, fill)
    rows = RowMeta(m)
    rows.write(positions, owners, m)
    spec = ops.AttnSpec(q_heads=nq, window=case["window"], scale=ops.default_scale(hd), m=m, causal=True, seq=None,
                        args=rows, softcap=case["softcap"])
    torch.cuda.synchronize()
    y, ko, vo = _outputs(case, m)
    return {"kind": case["kind"], "ops": ops, "pool": pool, "rows": rows, "spec": spec, "m": m, "q": q, "k": k, "v": v,
            "y": y, "ko": ko, "vo": vo, "keep": fill}


def _prepare_plain(case, seed):
    nq, nkv, hd = MODELS[case["model"]]
    page = case["page"]
    tables = [torch.tensor(p, device="cuda") for p in _pages(case)]
    slots = sum(len(p) for p in tables) * page
    positions, owners = _rows(case)
    m = len(owners)
    q, k, v = _new(case, seed, m)
    cache = {"k": torch.zeros(slots, nkv, hd, dtype=torch.float8_e4m3fn, device="cuda"),
             "v": torch.zeros(slots, nkv, hd, dtype=torch.float8_e4m3fn, device="cuda"),
             "ks": torch.zeros(slots, nkv, dtype=torch.uint8, device="cuda"),
             "vs": torch.zeros(slots, nkv, dtype=torch.uint8, device="cuda")}
    for s, t0, kc, vc in _contents(case, seed, k, v):
        pos = torch.arange(t0, t0 + kc.shape[0], device="cuda")
        _plain_store(cache, tables[s][pos // page] * page + pos % page, kc, vc)
    pos = torch.tensor(positions, device="cuda")
    table = torch.zeros(len(tables), max(len(t) for t in tables), dtype=torch.int64, device="cuda")
    for s, t in enumerate(tables):
        table[s, :len(t)] = t
    own_t = torch.tensor(owners, device="cuda")
    slot = table[own_t, pos // page] * page + pos % page
    torch.cuda.synchronize()
    return {"kind": case["kind"], "case": case, "seqs": _sequences(case), "tables": tables, "cache": cache,
            "slot": slot, "q": q, "k": k, "v": v}


# ---------------------------------------------------------------- one pass


def run(state):
    if "ops" not in state:
        return _run_plain(state)
    ops, pool, rows, m = state["ops"], state["pool"], state["rows"], state["m"]
    if state["kind"] == "store":
        ops.kv_store(state["k"], state["v"], pool, 0, m, rows)
    elif state["kind"] == "attn":
        ops.attn(state["q"], pool, 0, state["y"], state["spec"])
        return {"y": state["y"]}
    else:
        ops.kv_store_attn(state["k"], state["v"], state["q"], pool, 0, state["y"], state["spec"])
    ops.kv_load(state["ko"], state["vo"], pool, 0, m, rows)
    out = {"k": state["ko"], "v": state["vo"]}
    return out if state["kind"] == "store" else {"y": state["y"], **out}


def _plain_quantise(x):
    """Codes and biased scale exponents of head vectors [..., head_dim]."""
    x = x.float()
    bits = x.abs().amax(-1).view(torch.int32)
    b = ((bits >> 23) - 8 + ((bits & 0x7FFFFF) > 0x600000).int()).clamp(1, 254)
    inv = ((254 - b) << 23).view(torch.float32)
    return (x * inv[..., None]).to(torch.float8_e4m3fn), b.to(torch.uint8)


def _plain_values(codes, b):
    return codes.float() * (b.int() << 23).view(torch.float32)[..., None]


def _plain_store(cache, slot, k, v):
    for name, x in (("k", k), ("v", v)):
        codes, b = _plain_quantise(x)
        cache[name].view(torch.uint8)[slot] = codes.view(torch.uint8)
        cache[name + "s"][slot] = b


def _plain_load(cache, slot, name):
    codes = cache[name].view(torch.uint8)[slot].view(torch.float8_e4m3fn)
    return _plain_values(codes, cache[name + "s"][slot])


def _run_plain(state):
    case, cache, slot = state["case"], state["cache"], state["slot"]
    dt = DTYPES[case["y"]]
    if state["kind"] != "attn":
        _plain_store(cache, slot, state["k"], state["v"])
    out = {}
    if state["kind"] != "store":
        page, at, ys = case["page"], 0, []
        for s, (c, n) in enumerate(state["seqs"]):
            first = max(0, c + 1 - case["window"]) if case["window"] else 0
            t = torch.arange(first, c + n, device="cuda")
            at_slot = state["tables"][s][t // page] * page + t % page
            k, v = (_plain_load(cache, at_slot, name).transpose(0, 1).contiguous() for name in ("k", "v"))
            ys.append(_attend(state["q"][at:at + n].float(), k, v, first, c, case["window"], case["softcap"]).to(dt))
            at += n
        out["y"] = torch.cat(ys)
    if state["kind"] != "attn":
        out["k"], out["v"] = (_plain_load(cache, slot, name).to(dt) for name in ("k", "v"))
    return out


def _attend(q, k, v, t0, first, window, softcap):
    """Causal attention of q [m, heads, hd] at positions first.. over k and v
    [kv_heads, n, hd], whose first key is at position t0, in q's type."""
    m, nq, hd = q.shape
    nkv, n, _ = k.shape
    g = nq // nkv
    kt = k.transpose(1, 2).contiguous()
    t = t0 + torch.arange(n, device=q.device)
    out = torch.empty(m, nq, hd, dtype=q.dtype, device=q.device)
    step = max(16, (1 << 28) // max(1, nq * n))
    for r in range(0, m, step):
        b = min(step, m - r)
        qr = q[r:r + b].reshape(b, nkv, g, hd).permute(1, 2, 0, 3).reshape(nkv, g * b, hd).contiguous()
        s = torch.matmul(qr, kt) * (1.0 / math.sqrt(hd))
        if softcap:
            s = softcap * torch.tanh(s / softcap)
        p = first + r + torch.arange(b, device=q.device)
        mask = t[None, :] > p[:, None]
        if window:
            mask |= t[None, :] <= p[:, None] - window
        s = s.view(nkv, g, b, n).masked_fill(mask, -math.inf)
        s = torch.exp(s - s.amax(-1, keepdim=True))
        o = torch.matmul(s.view(nkv, g * b, n), v) / s.sum(-1).view(nkv, g * b, 1)
        out[r:r + b] = o.view(nkv, g, b, hd).permute(2, 0, 1, 3).reshape(b, nq, hd)
    return out


# --------------------------------------------------------- in 64 bits


def _pow2(e):
    """2^e in f64, by its exponent field (torch's ldexp takes a power, which is not exact)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _stored64(x):
    """The values that the cache holds for head vectors x, from the format's definition."""
    x = x.double()
    mant, e = torch.frexp(x.abs().amax(-1, keepdim=True) / 448.0)
    e = torch.where(mant == 0.5, e - 1, e).clamp(min=-126)
    t = x * _pow2(-e)
    _, te = torch.frexp(t)
    quantum = _pow2((te - 1).clamp(min=-6) - 3)
    return torch.round(t / quantum) * quantum * _pow2(e)


def exact(case, seed):
    positions, owners = _rows(case)
    m = len(owners)
    q, k, v = _new(case, seed, m)
    ks, vs = _stored64(k), _stored64(v)
    out = {}
    if case["kind"] != "store":
        seqs = _sequences(case)
        nq, _, hd = MODELS[case["model"]]
        if 4 * nq * hd * sum(n * (c + n) for c, n in seqs) > 2e13:
            return None
        at, ys = 0, []
        for s, (c, n) in enumerate(seqs):
            kk, vv = ks[at:at + n], vs[at:at + n]
            if c:
                kc, vc = _cached(case, seed, s, c)
                kk, vv = torch.cat([_stored64(kc), kk]), torch.cat([_stored64(vc), vv])
            kk, vv = (x.transpose(0, 1).contiguous() for x in (kk, vv))
            ys.append(_attend64(q[at:at + n].double(), kk, vv, c, case["window"], case["softcap"]))
            at += n
        out["y"] = torch.cat(ys)
    if case["kind"] != "attn":
        out["k"], out["v"] = ks, vs
    return out


def _attend64(q, k, v, first, window, softcap):
    """The definition in 64 bits, one query head at a time."""
    m, nq, hd = q.shape
    nkv, n, _ = k.shape
    out = torch.empty_like(q)
    t = torch.arange(n, device=q.device)
    for h in range(nq):
        kv = h // (nq // nkv)
        for r in range(0, m, 1024):
            b = min(1024, m - r)
            s = torch.mm(q[r:r + b, h], k[kv].t().contiguous()) / math.sqrt(hd)
            if softcap:
                s = softcap * torch.tanh(s / softcap)
            p = first + torch.arange(r, r + b, device=q.device)
            seen = (t[None, :] <= p[:, None]) & ((t[None, :] > p[:, None] - window) if window else True)
            s = torch.where(seen, s, torch.full_like(s, -math.inf))
            w = torch.softmax(s, -1)
            out[r:r + b, h] = torch.mm(w, v[kv])
    return out


# ------------------------------------------------------------------- work


def work(case):
    nq, nkv, hd = MODELS[case["model"]]
    seqs = _sequences(case)
    m = sum(n for _, n in seqs)
    vec = hd + 1  # a head vector's codes and its scale
    nbytes = flops = 0
    if case["kind"] != "attn":  # sources read; codes written and read; values written
        nbytes += 2 * m * nkv * (hd * (BYTES[case["x"]] + BYTES[case["y"]]) + 2 * vec)
        flops += 8 * m * nkv * hd
    if case["kind"] != "store":
        w = case["window"]
        keys = pairs = 0
        for c, n in seqs:
            keys += min(c, w - 1) + n if w else c + n
            if w:
                pairs += sum(min(w, c + i + 1) for i in range(n))
            else:
                pairs += n * c + n * (n + 1) // 2
        nbytes += 2 * keys * nkv * vec + m * nq * hd * (BYTES[case["x"]] + BYTES[case["y"]])
        flops += 4 * pairs * nq * hd
    return {"bytes": nbytes, "flops": flops}
