"""What is measured of the 8-bit KV cache and of eviction from it: the listed cases, their inputs, a plain form of
every operator in elementary torch operations, and an exact form in 64 bits.

The cache holds K and V in 8 bits (int8, or fp8 e4m3) with one scale for each block of 32 tokens and kv head, for K
and for V; tokens of a block that is not complete and committed stay in fp16 (the tail). Its operators:

  attend   attention of the last m tokens (one decoded token, or a round of drafts) over the cache
  prefill  the same for a prompt chunk
  append   storing new tokens (and turning complete blocks into 8 bits), read back as the values the cache stands for
  weights  each cached key's attention weight, summed over the m tokens and the query heads of its kv head, on top of
           an older sum that decays
  evict    keeping the first `sink`, the last `recent` and the heaviest keys of each kv head up to a budget, and moving
           them into a smaller cache
"""
import math

import torch

own = False

BLOCK = 32
QMAX = {"int8": 127.0, "e4m3": 448.0}


def _case(kind, name, **kw):
    base = {"kind": kind, "fmt": "int8", "q_heads": 32, "kv_heads": 8, "head_dim": 64}
    base.update(kw)
    if name:
        base["name"] = name
    return base


def listed():
    wide = {"q_heads": 16, "kv_heads": 4, "head_dim": 128}   # the engine's model; the other is the benchmark's geometry
    return [
        # one decoded token early in a chat: the smallest call, all latency
        _case("attend", "decode_short", ctx=777, m=1, window=0, gate=False),
        # one decoded token over a long document: every cached byte read once
        _case("attend", "decode_long", ctx=100003, m=1, window=0, gate=False),
        # the engine's own verify round (8 tokens, gated output)
        _case("attend", "verify_gated", fmt="e4m3", ctx=32768, m=8, window=0, gate=True, **wide),
        # the benchmark's longest round: 16 drafts over 131072 cached tokens
        _case("attend", "verify_long", ctx=131072, m=16, window=0, gate=False),
        # a prompt chunk in a sliding-window layer
        _case("prefill", "prefill_window", tokens=2048, ctx=4096, window=256, **wide),
        # a ragged chunk of a long prompt in a full layer
        _case("prefill", "prefill_long", fmt="e4m3", tokens=1999, ctx=30001, window=0, **wide),
        # a round's drafts, the block before them complete and committed
        _case("append", "append_drafts", ctx=32773, n=16, draft=True, lag=13),
        # the engine's largest prompt chunk
        _case("append", "append_prompt", fmt="e4m3", ctx=115200, n=7680, draft=False, lag=0, **wide),
        # weights of one decoded token over a long document
        _case("weights", "weights_decode", ctx=131072, m=1, decay=1.0),
        # weights of the last 32 tokens of a prompt (an observation window)
        _case("weights", "weights_prompt", fmt="e4m3", ctx=20000, m=32, decay=0.95, **wide),
        # a long context cut to a quarter
        _case("evict", "evict_long", len=131072, budget=32768, sink=4, recent=256),
        # a short ragged one, in the engine's geometry
        _case("evict", "evict_short", fmt="e4m3", len=5003, budget=2047, sink=1, recent=100, **wide),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "prefill", "append", "weights", "evict"])
    fmt = rng.choice(["int8", "e4m3"])
    q_heads, kv_heads, head_dim = rng.choice([(32, 8, 64), (16, 4, 128), (8, 2, 128), (12, 3, 64), (24, 6, 64)])
    case = _case(kind, None, fmt=fmt, q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim)
    if kind == "attend":
        m = rng.choice([1, 1, 2, 3, 4, 5, 7, 8, 9, 12, 16, 24, 32])
        ctx = _log_int(rng, 32, 131072)
        window = 0 if rng.random() < 0.7 else max(m, _log_int(rng, 64, 2048))
        case.update(ctx=ctx, m=m, window=window, gate=rng.random() < 0.5)
    elif kind == "prefill":
        case.update(tokens=_log_int(rng, 40, 2048), ctx=_log_int(rng, 32, 28000),
                    window=0 if rng.random() < 0.6 else _log_int(rng, 64, 1024))
    elif kind == "append":
        draft = rng.random() < 0.5
        case.update(ctx=_log_int(rng, 64, 32768), n=rng.randint(1, 32) if draft else _log_int(rng, 1, 7680), draft=draft,
                    lag=rng.randint(0, 20))
    elif kind == "weights":
        case.update(ctx=_log_int(rng, 32, 131072), m=rng.choice([1, 1, 2, 4, 8, 13, 16, 32]),
                    decay=rng.choice([1.0, 0.95, 0.5]))
    else:
        length = _log_int(rng, 200, 131072)
        sink, recent = rng.randint(0, 8), rng.randint(32, 64)
        case.update(len=length, sink=sink, recent=recent, budget=rng.randint(sink + recent, length))
    return case


# ------------------------------------------------------------------ inputs (the same for every form)
def _normal(gen, *shape, scale=1.0):
    return (torch.randn(*shape, generator=gen, device="cuda") * scale).half()


def _cache_rows(gen, n, heads, dim):
    """K rows with a few strong channels, as a key projection has them, and V rows."""
    channel = torch.exp(0.5 * torch.randn(1, heads, dim, generator=gen, device="cuda"))
    k = (torch.randn(n, heads, dim, generator=gen, device="cuda") * channel).half()
    return k, _normal(gen, n, heads, dim)


def _quantise(x, fmt):
    """Blocks of 32 tokens [n][heads][dim] in 8 bits: (values [n / 32][heads][32][dim], scales [n / 32][heads]); the
    scale is absmax over the block and head / 127 (448 for e4m3), 1 for a block of zeros."""
    n, heads, dim = x.shape
    b = x.float().reshape(n // BLOCK, BLOCK, heads, dim).transpose(1, 2)
    top = b.abs().amax(dim=(2, 3))
    # a float32 tensor as the divisor: a Python number would be multiplied by its rounded reciprocal
    scale = torch.where(top > 0, top / torch.full_like(top, QMAX[fmt]), torch.ones_like(top))
    y = b / scale[:, :, None, None]
    q = torch.round(y).clamp(-127, 127).to(torch.int8) if fmt == "int8" else y.to(torch.float8_e4m3fn)
    return q, scale


def _values(q, scale):
    """The float32 values [n][heads][dim] that 8-bit blocks stand for."""
    v = q.float() * scale[:, :, None, None]
    return v.transpose(1, 2).reshape(-1, q.shape[1], q.shape[3])


def _lengths(case):
    """(tokens in all, committed tokens): the blocks complete among the committed ones are in 8 bits."""
    kind = case["kind"]
    if kind in ("attend", "weights"):
        return case["ctx"] + case["m"], case["ctx"]
    if kind == "prefill":
        return case["ctx"] + case["tokens"], case["ctx"] + case["tokens"]
    if kind == "evict":
        return case["len"], case["len"]
    # append: the tokens from `lag` before the new ones on are in the tail when the call is made
    return case["ctx"], max(0, case["ctx"] - case["lag"])


def _inputs(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    heads, dim, qh = case["kv_heads"], case["head_dim"], case["q_heads"]
    total, committed = _lengths(case)
    k, v = _cache_rows(gen, total, heads, dim)
    sealed = committed // BLOCK * BLOCK
    d = {"k": k, "v": v, "total": total, "committed": committed, "sealed": sealed}
    kind = case["kind"]
    if kind in ("attend", "weights", "prefill"):
        rows = case["tokens"] if kind == "prefill" else case["m"]
        d["q"] = _normal(gen, rows, qh, dim, scale=1.2)
    if case.get("gate"):
        d["gate"] = _normal(gen, case["m"], qh)
    if kind == "append":
        d["k_new"], d["v_new"] = _cache_rows(gen, case["n"], heads, dim)
    if kind in ("weights", "evict"):
        # sums of softmax weights so far: most keys little, some much
        w = torch.rand(heads, total, generator=gen, device="cuda")
        d["prev"] = w.pow(8) * 4.0
    return d


def _blocks(case, d):
    s = d["sealed"]
    k8, ks = _quantise(d["k"][:s], case["fmt"])
    v8, vs = _quantise(d["v"][:s], case["fmt"])
    return {"k8": k8, "ks": ks, "v8": v8, "vs": vs, "k_tail": d["k"][s:], "v_tail": d["v"][s:]}


def prepare(case, seed):
    d = _inputs(case, seed)
    blocks = _blocks(case, d)
    state = {"case": case, "total": d["total"], "sealed": d["sealed"]}
    for name in ("q", "gate", "k_new", "v_new", "prev"):
        if name in d:
            state[name] = d[name]
    if case["kind"] == "weights":
        state["lse"] = _softmax_lse(case, state["q"], _cached(blocks)[0])
    if not own:
        state.update(blocks)
        return state
    import sys

    if "lfm3-1.7b-mi50_b200" not in sys.path:
        sys.path.insert(0, "lfm3-1.7b-mi50_b200")
    import lfm3attn as la

    mode = la.MODE_I8BLK if case["fmt"] == "int8" else la.MODE_E4M3BLK
    room = d["total"] + (case["n"] if case["kind"] == "append" else 0)
    cache = la.LayerCache8(mode, case["kv_heads"], case["head_dim"], room)
    c = d["committed"]
    if c:
        cache.append(d["k"][:c].contiguous(), d["v"][:c].contiguous())
    if d["total"] > c:
        cache.append(d["k"][c:].contiguous(), d["v"][c:].contiguous(), draft=True)
    state["cache"] = cache
    if case["kind"] in ("attend", "prefill"):
        state["workspace"] = cache.workspace(state["q"].shape[0], case["q_heads"])
    if case["kind"] == "evict":
        state["dst"] = la.LayerCache8(mode, case["kv_heads"], case["head_dim"], case["budget"])
    return state


# ------------------------------------------------------------------ the plain form
def _cached(s):
    """Every cached token's K and V [n][heads][dim] as float32."""
    k, v = s["k_tail"].float(), s["v_tail"].float()
    if s["k8"].shape[0]:
        k, v = torch.cat([_values(s["k8"], s["ks"]), k]), torch.cat([_values(s["v8"], s["vs"]), v])
    return k, v


def _scores(case, q, k):
    """Scores [heads][tokens x group][keys]; keys after a token, or `window` or more before it, are masked."""
    t, qh, dim = q.shape
    n, heads, _ = k.shape
    rows = q.float().reshape(t, heads, qh // heads, dim).permute(1, 0, 2, 3).reshape(heads, -1, dim)
    s = torch.matmul(rows, k.permute(1, 2, 0)) / math.sqrt(dim)
    at = (n - t + torch.arange(t, device=q.device)).repeat_interleave(qh // heads)[:, None]
    key = torch.arange(n, device=q.device)[None, :]
    hidden = key > at
    if case.get("window"):
        hidden = hidden | (key <= at - case["window"])
    return s.masked_fill_(hidden, float("-inf"))


def _rows_back(x, t, qh):
    heads = x.shape[0]
    return x.reshape(heads, t, qh // heads, -1).permute(1, 0, 2, 3).reshape(t, qh, -1)


def _softmax_lse(case, q, k):
    s = _scores(case, q, k)
    top = s.amax(dim=-1, keepdim=True)
    lse = top + torch.log(torch.exp(s - top).sum(dim=-1, keepdim=True))
    return _rows_back(lse, q.shape[0], q.shape[1])[:, :, 0].contiguous()


def _attend_plain(s):
    case, q = s["case"], s["q"]
    k, v = _cached(s)
    x = _scores(case, q, k)
    top = x.amax(dim=-1, keepdim=True)
    p = torch.exp(x - top)
    total = p.sum(dim=-1, keepdim=True)
    o = torch.matmul(p, v.permute(1, 0, 2)) / total
    out = _rows_back(o, q.shape[0], q.shape[1])
    if "gate" in s:
        out = out * torch.sigmoid(s["gate"].float())[:, :, None]
    got = {"out": out.half()}
    if case["kind"] == "attend":
        got["lse"] = _rows_back(top + torch.log(total), q.shape[0], q.shape[1])[:, :, 0].contiguous()
    return got


def _append_plain(s):
    case = s["case"]
    k, v = torch.cat([s["k_tail"], s["k_new"]]), torch.cat([s["v_tail"], s["v_new"]])
    end = case["ctx"] if case["draft"] else case["ctx"] + case["n"]
    full = max(0, end // BLOCK * BLOCK - s["sealed"])
    got = {}
    for name, x in (("k", k), ("v", v)):
        done = _values(*_quantise(x[:full], case["fmt"])).half() if full else x[:0]
        got[name] = torch.cat([done, x[full:]])
    return got


def _weights_plain(s):
    case, q = s["case"], s["q"]
    k, _ = _cached(s)
    heads, qh = case["kv_heads"], case["q_heads"]
    lse = s["lse"].reshape(-1, heads, qh // heads).permute(1, 0, 2).reshape(heads, -1, 1)
    return {"weights": s["prev"] * case["decay"] + torch.exp(_scores(case, q, k) - lse).sum(dim=1)}


def _keep_plain(w, case):
    """[heads][budget] kept positions, ascending: the first `sink`, the last `recent`, and of the others the heaviest
    (of equal ones the first)."""
    heads, n = w.shape
    sink, recent, budget = case["sink"], case["recent"], case["budget"]
    always = torch.zeros(n, dtype=torch.bool, device=w.device)
    always[:sink] = True
    always[n - recent:] = True
    key = torch.where(always[None, :], torch.full_like(w, float("inf")), w)
    order = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :budget]
    return torch.sort(order, dim=1).values


def _evict_plain(s):
    case = s["case"]
    w = s["prev"]
    keep = _keep_plain(w, case)
    k, v = _cached(s)
    got = {"keep": keep.to(torch.int32), "weights": torch.gather(w, 1, keep)}
    full = case["budget"] // BLOCK * BLOCK
    index = keep.t()[:, :, None].expand(-1, -1, case["head_dim"])
    for name, x in (("k", k), ("v", v)):
        x = torch.gather(x, 0, index)
        done = _values(*_quantise(x[:full], case["fmt"])).half() if full else x[:0].half()
        got[name] = torch.cat([done, x[full:].half()])
    return got


def run(state):
    case = state["case"]
    kind = case["kind"]
    if not own:
        if kind in ("attend", "prefill"):
            return _attend_plain(state)
        return {"append": _append_plain, "weights": _weights_plain, "evict": _evict_plain}[kind](state)
    cache = state["cache"]
    if kind == "attend":
        q = state["q"]
        lse = torch.empty(q.shape[0], q.shape[1], dtype=torch.float32, device=q.device)
        out = cache.verify(q, case["ctx"], window=case["window"], gate=state.get("gate"), lse=lse,
                           workspace=state["workspace"])
        return {"out": out, "lse": lse}
    if kind == "prefill":
        return {"out": cache.prefill(state["q"], case["ctx"], window=case["window"], workspace=state["workspace"])}
    if kind == "append":
        cache.length, cache.sealed = case["ctx"], state["sealed"]   # as before the call, when the pass is repeated
        cache.append(state["k_new"], state["v_new"], draft=case["draft"])
        k, v = cache.read(state["sealed"], case["ctx"] + case["n"] - state["sealed"])
        return {"k": k, "v": v}
    if kind == "weights":
        return {"weights": cache.key_weights(state["q"], state["lse"], case["ctx"], prev=state["prev"],
                                             decay=case["decay"])}
    keep, weights = cache.evict(state["prev"], case["budget"], case["sink"], case["recent"], dst=state["dst"])
    k, v = state["dst"].read(0, case["budget"])
    return {"keep": keep, "weights": weights, "k": k, "v": v}


# ------------------------------------------------------------------ the work that cannot be left out
def _visible(t, n, window):
    """Pairs of a token and a key it sees, t tokens at the end of n."""
    pairs = 0
    for i in range(t):
        seen = n - t + i + 1
        pairs += min(seen, window) if window else seen
    return pairs


def work(case):
    heads, dim, qh = case["kv_heads"], case["head_dim"], case["q_heads"]
    total, committed = _lengths(case)
    kind = case["kind"]
    if kind in ("attend", "prefill"):
        t = case["m"] if kind == "attend" else case["tokens"]
        first = max(0, total - t - case["window"] + 1) if case["window"] else 0
        sealed = max(0, committed // BLOCK * BLOCK - first)
        tail = total - max(first, committed // BLOCK * BLOCK)
        by = heads * (sealed * dim * 2 + sealed // BLOCK * 8 + tail * dim * 4) + t * qh * dim * 4
        by += t * qh * 4 if kind == "attend" else 0
        return {"bytes": by, "flops": 4 * dim * qh * _visible(t, total, case["window"])}
    if kind == "append":
        old = total - committed // BLOCK * BLOCK
        n = case["n"] + old
        end = case["ctx"] if case["draft"] else case["ctx"] + case["n"]
        full = max(0, end // BLOCK * BLOCK - committed // BLOCK * BLOCK)
        # new rows and the old tail read, what becomes 8 bits written, the rest written in fp16, the values returned
        by = heads * dim * 2 * (2 * n + full + 2 * min(n - full, case["n"]) + 2 * n)
        return {"bytes": by, "flops": 4 * n * heads * dim}
    if kind == "weights":
        sealed = committed // BLOCK * BLOCK
        by = heads * (sealed * dim + sealed // BLOCK * 4 + (total - sealed) * dim * 2 + total * 8)
        by += case["m"] * qh * (dim * 2 + 4)
        return {"bytes": by, "flops": 2 * dim * qh * _visible(case["m"], total, 0)}
    n, keep = case["len"], case["budget"]
    # the weights read; each kept token's K and V read and written in 8 bits, its position and weight; the values returned
    by = heads * (n * 4 + keep * (2 * dim * 2 + 8) + keep * 2 * dim * 2)
    return {"bytes": by, "flops": heads * (n + 8 * keep * dim)}


# ------------------------------------------------------------------ in 64 bits, from the definitions
def _exact_blocks(x, fmt):
    """What blocks of 32 rows [n][heads][dim] come back as from 8 bits. By definition the scale, the quotient that is
    rounded to 8 bits and the value it stands for are float32, so that ties fall the same way everywhere."""
    n, heads, dim = x.shape
    b = x.double().view(n // BLOCK, BLOCK, heads, dim)
    top = b.abs().amax(dim=3, keepdim=True).amax(dim=1, keepdim=True)
    scale = (top / QMAX[fmt]).float().double()
    scale[scale == 0] = 1.0
    y = (b / scale).float().double()
    if fmt == "int8":
        y = torch.round(y).clamp(-127, 127)
    else:
        # 3 bits after the leading one; below 2^-6 a grid of 2^-9
        step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
        y = (torch.round(y / step) * step).clamp(-448, 448)
    return (y * scale).float().double().view(n, heads, dim)


def _exact_cached(case, d):
    s = d["sealed"]
    out = []
    for x in (d["k"], d["v"]):
        done = _exact_blocks(x[:s], case["fmt"]) if s else x[:0].double()
        out.append(torch.cat([done, x[s:].double()]))
    return out


def exact(case, seed):
    d = _inputs(case, seed)
    kind = case["kind"]
    heads, dim, qh = case["kv_heads"], case["head_dim"], case["q_heads"]
    group = qh // heads
    if kind == "append":
        end = case["ctx"] if case["draft"] else case["ctx"] + case["n"]
        full = max(0, end // BLOCK * BLOCK - d["sealed"])
        got = {}
        for name in ("k", "v"):
            x = torch.cat([d[name][d["sealed"]:], d[name + "_new"]])
            done = _exact_blocks(x[:full], case["fmt"]) if full else x[:0].double()
            got[name] = torch.cat([done, x[full:].double()])
        return got
    k, v = _exact_cached(case, d)
    n = k.shape[0]
    if kind == "evict":
        w = d["prev"]
        keeps = []
        for h in range(heads):
            mid = sorted(range(case["sink"], n - case["recent"]), key=lambda i, r=w[h].tolist(): (-r[i], i))
            mid = mid[:case["budget"] - case["sink"] - case["recent"]]
            keeps.append(sorted(list(range(case["sink"])) + mid + list(range(n - case["recent"], n))))
        keep = torch.tensor(keeps, device=w.device)
        full = case["budget"] // BLOCK * BLOCK
        got = {"keep": keep.to(torch.int32), "weights": torch.stack([w[h][keep[h]] for h in range(heads)]).double()}
        for name, x in (("k", k), ("v", v)):
            x = torch.stack([x[keep[h], h] for h in range(heads)], dim=1)
            done = _exact_blocks(x[:full], case["fmt"]) if full else x[:0]
            got[name] = torch.cat([done, x[full:]])
        return got
    q = d["q"].double()
    t = q.shape[0]
    pos = torch.arange(n, device=q.device)
    window = case.get("window", 0)
    outs, lses, sums = [], [], []
    lse_in = _softmax_lse(case, d["q"], _cached(_blocks(case, d))[0]).double() if kind == "weights" else None
    for h in range(heads):
        kh, vh = k[:, h], v[:, h]
        qs = q[:, h * group:(h + 1) * group].reshape(t * group, dim)
        x = (qs @ kh.T) * dim ** -0.5
        mine = (n - t + torch.arange(t, device=q.device)).repeat_interleave(group)
        seen = pos[None] <= mine[:, None]
        if window:
            seen &= pos[None] > mine[:, None] - window
        if kind == "weights":
            e = torch.exp(x - lse_in[:, h * group:(h + 1) * group].reshape(-1, 1))
            sums.append(torch.where(seen, e, torch.zeros_like(e)).sum(0))
            continue
        x[~seen] = -math.inf
        z = torch.logsumexp(x, dim=1)
        outs.append((torch.exp(x - z[:, None]) @ vh).view(t, group, dim))
        lses.append(z.view(t, group))
    if kind == "weights":
        return {"weights": d["prev"].double() * case["decay"] + torch.stack(sums)}
    out = torch.cat(outs, dim=1)
    if "gate" in d:
        out = out / (1 + torch.exp(-d["gate"].double()))[:, :, None]
    return {"out": out, "lse": torch.cat(lses, dim=1)} if kind == "attend" else {"out": out}
