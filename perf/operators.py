"""What the serving operators are measured on: appending to a paged KV cache, attention over it, drawing tokens from logits.

With ``own`` false `run` computes each operator in its plain form (elementary torch operations); with ``own`` true it makes
the calls a user makes of the library: ``kv_append_dev``, ``attn_pages_dev`` and ``sample_dev`` of ``CudaWeightAccel``.

The cache: pages of `page` tokens, ``[n_pages][kv_heads][page][hd]`` for k and for v, in f16, or in e4m3 with one
power-of-two scale for each page and head. A batch: ``row0[n_seq + 1]`` (first new row of each sequence), ``ctx[n_seq]``
(tokens cached before; below zero an idle slot), ``table[n_seq][pages_ld]`` (page ids).
"""
import math

import numpy as np
import torch

own = False

_MOST_ROWS_HD = 8192 * 48 * 128        # of an append: rows x heads (q, k and v) x head size
_MOST_CACHED = 64 * 16384 * 8 * 128    # of attention: sequences x longest context x kv heads x head size
_MOST_PAIRS = 4.5e6 * 32 * 128         # of attention: (query row, token) pairs x heads x head size


def listed():
    a = dict(op="append", heads=32, kv_heads=8, hd=128, page=64, rope="halves", theta=1e6, norm=True, idle=0)
    t = dict(op="attn", heads=32, kv_heads=8, hd=128, page=64, window=0, idle=0)
    return [
        # one decoded token of one user: a launch is all there is
        dict(a, name="append 1 token", kv="e4m3", n_seq=1, new_lo=1, new_hi=1, ctx_lo=777, ctx_hi=777),
        # a decode step of a full batch, wide heads, the cache in 16 bits, two slots of the captured batch idle
        dict(a, name="append 64 seqs f16", kv="f16", n_seq=64, new_lo=1, new_hi=1, ctx_lo=200, ctx_hi=1000, heads=16, kv_heads=8,
             hd=256, idle=2),
        # prompts of five users entering the cache
        dict(a, name="append prompts", kv="e4m3", n_seq=5, new_lo=300, new_hi=4000, ctx_lo=0, ctx_hi=100),
        # one user at the start of a chat
        dict(t, name="attn 1 x 300", kv="e4m3", n_seq=1, new_lo=1, new_hi=1, ctx_lo=300, ctx_hi=300),
        # one user with a book in the context
        dict(t, name="attn 1 x 131071", kv="e4m3", n_seq=1, new_lo=1, new_hi=1, ctx_lo=131071, ctx_hi=131071),
        # a full batch of chats of all lengths, three slots idle
        dict(t, name="attn 64 ragged", kv="e4m3", n_seq=61, new_lo=1, new_hi=1, ctx_lo=500, ctx_hi=16384, idle=3),
        # speculative decoding: five rows of eight users to verify
        dict(t, name="attn verify 8 x 5 f16", kv="f16", n_seq=8, new_lo=5, new_hi=5, ctx_lo=1000, ctx_hi=5000, page=32),
        # a chunk of a long prompt
        dict(t, name="attn prompt chunk", kv="e4m3", n_seq=1, new_lo=512, new_hi=512, ctx_lo=8000, ctx_hi=8000),
        # the local layers of a model with wide heads
        dict(t, name="attn window 1024 f16", kv="f16", n_seq=24, new_lo=1, new_hi=3, ctx_lo=100, ctx_hi=9000, heads=8, kv_heads=4,
             hd=256, page=16, window=1024),
        dict(op="sample", name="sample 1 chat", rows=1, n=151936, how="chat"),
        dict(op="sample", name="sample 64 mixed", rows=64, n=151936, how="mixed"),
        dict(op="sample", name="sample 16 nucleus", rows=16, n=262147, how="nucleus"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "attn", "attn", "sample"])
    if op == "sample":
        return dict(op=op, rows=_log(rng, 1, 64), n=_log(rng, 1000, 262147), how=rng.choice(["chat", "mixed", "nucleus", "open"]))
    kv_heads = rng.choice([1, 2, 4, 5, 8, 16])
    c = dict(op=op, kv=rng.choice(["f16", "e4m3"]), kv_heads=kv_heads, heads=kv_heads * rng.choice([1, 2, 3, 4, 7, 8]),
             hd=rng.choice([64, 96, 128, 192, 256]), page=rng.choice([16, 32, 64, 128]), idle=rng.choice([0, 0, 1, 2]))
    if op == "append":
        c.update(rope=rng.choice(["none", "halves", "adjacent"]), theta=rng.choice([1e4, 5e5, 1e6]), norm=rng.random() < 0.5,
                 n_seq=_log(rng, 1, 64), new_lo=1, new_hi=rng.choice([1, 1, 5, _log(rng, 1, 4096)]), ctx_lo=0, ctx_hi=_log(rng, 1, 1500))
        while sum(_spread(c["new_lo"], c["new_hi"], c["n_seq"])) * (c["heads"] + 2 * kv_heads) * c["hd"] > _MOST_ROWS_HD // 2:
            c["new_hi"] = max(1, c["new_hi"] // 2)
            c["n_seq"] = max(1, c["n_seq"] * 3 // 4)
        return c
    c.update(window=rng.choice([0, 0, 0, _log(rng, 16, 4096)]), n_seq=_log(rng, 1, 64), new_lo=1,
             new_hi=rng.choice([1, 1, 1, 2, 5, 8, _log(rng, 8, 512)]), ctx_lo=0, ctx_hi=_log(rng, 1, 100000))
    while (c["n_seq"] * (c["ctx_hi"] + c["new_hi"]) * kv_heads * c["hd"] > _MOST_CACHED // 2
           or c["n_seq"] * c["new_hi"] * (c["ctx_hi"] + c["new_hi"]) * c["heads"] * c["hd"] > _MOST_PAIRS):
        c["ctx_hi"] = max(1, c["ctx_hi"] * 2 // 3)
        c["new_hi"] = max(1, c["new_hi"] * 3 // 4)
        c["n_seq"] = max(1, c["n_seq"] * 4 // 5)
    return c


def _spread(lo, hi, n):
    """n whole numbers from lo to hi, evenly over their logarithm, in a fixed mixed order."""
    if n == 1:
        return [hi]
    v = [int(round(math.exp(math.log(lo + 1) + (math.log(hi + 1) - math.log(lo + 1)) * i / (n - 1)))) - 1 for i in range(n)]
    order = np.random.RandomState(n).permutation(n)
    return [v[i] for i in order]


def _lengths(c):
    """(new rows, tokens cached before) of every slot; an idle slot has one row and ctx -1."""
    new = _spread(c["new_lo"], c["new_hi"], c["n_seq"]) + [1] * c["idle"]
    ctx = _spread(c["ctx_lo"], c["ctx_hi"], c["n_seq"]) + [-1] * c["idle"]
    return new, ctx


def work(case):
    c = case
    if c["op"] == "sample":
        return {"bytes": 4.0 * c["rows"] * c["n"], "flops": 4.0 * c["rows"] * c["n"]}
    new, ctx = _lengths(c)
    el = 2 if c["kv"] == "f16" else 1
    live = [(n, x) for n, x in zip(new, ctx) if x >= 0]
    rows = sum(n for n, _ in live)
    if c["op"] == "append":
        return {"bytes": float(rows * c["hd"] * (4 * (2 * c["heads"] + 2 * c["kv_heads"]) + 2 * el * c["kv_heads"])),
                "flops": float(rows * c["hd"] * 8 * (c["heads"] + c["kv_heads"]))}
    w = c["window"]
    cached = sum((x + n) - (max(0, x + 1 - w) if w else 0) for n, x in live)
    pairs = sum(min(x + i + 1, w) if w else x + i + 1 for n, x in live for i in range(n))
    return {"bytes": float(cached * c["kv_heads"] * c["hd"] * 2 * el + rows * c["heads"] * c["hd"] * 8),
            "flops": float(4 * pairs * c["heads"] * c["hd"])}


# ---------------------------------------------------------------- inputs

def _cache(c, n_pages, g):
    """A cache as appends have left it: keys and values near normal, some channels of the keys far larger than the rest."""
    shape = (n_pages, c["kv_heads"], c["page"], c["hd"])
    s = {}
    for name in ("k", "v"):
        x = torch.empty(shape, dtype=torch.float16, device="cuda").normal_(generator=g)
        if name == "k":
            x[..., 3::32] *= 4.0
        if c["kv"] == "f16":
            s[name], s[name + "_scale"] = x, None
            continue
        e = torch.randint(-8, -5, shape[:2], generator=g, device="cuda")
        scale = torch.exp2(e.float())
        codes = torch.empty(shape, dtype=torch.float8_e4m3fn, device="cuda")
        torch.clamp(x.mul_(64.0), -448.0, 448.0, out=x)
        codes.copy_(x)
        s[name], s[name + "_scale"] = codes, scale
    return s


def _batch(c, g):
    new, ctx = _lengths(c)
    need = [0 if x < 0 else -(-(x + n) // c["page"]) for n, x in zip(new, ctx)]
    n_pages, ld = sum(need) + 3, max(max(need), 1)
    ids = torch.randperm(n_pages, generator=g, device="cuda").int()
    at = torch.tensor(np.cumsum([0] + need[:-1]), device="cuda")[:, None] + torch.arange(ld, device="cuda")[None]
    table = ids[at.clamp(max=n_pages - 1)].contiguous()
    row0 = torch.tensor(np.cumsum([0] + new), dtype=torch.int32, device="cuda")
    touched = sum(0 if x < 0 else (x + n - 1) // c["page"] - x // c["page"] + 1 for n, x in zip(new, ctx))
    return dict(n_seq=len(new), rows=sum(new), n_pages=n_pages, pages_ld=ld, table=table, row0=row0, most=max(new), touched=touched,
                ctx=torch.tensor(ctx, dtype=torch.int32, device="cuda"), longest=max(x + n for n, x in zip(new, ctx) if x >= 0))


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    if c["op"] == "sample":
        rows, n = c["rows"], c["n"]
        x = torch.randn(rows, n, generator=g, device="cuda") * 2.5
        few = torch.randint(0, n, (rows, 40), generator=g, device="cuda")
        x.scatter_add_(1, few, torch.empty(rows, 40, device="cuda").exponential_(0.25, generator=g) + 4.0)
        r = torch.arange(rows, device="cuda")
        kind = {"chat": 0 * r, "nucleus": 0 * r + 1, "open": 0 * r + 2, "mixed": r % 4}[c["how"]]
        pick = lambda *v: torch.tensor(v, device="cuda")[kind].contiguous()  # noqa: E731
        wide = 0.7 + 0.5 * torch.rand(rows, generator=g, device="cuda")
        return dict(case=c, x=x, u=torch.rand(rows, generator=g, device="cuda"), temperature=torch.where(kind == 3, 0.0, wide),
                    top_k=pick(40, 0, 0, 0).int(), top_p=pick(0.95, 0.9, 1.0, 1.0).float(), min_p=pick(0.05, 0.0, 0.0, 0.0).float(),
                    ids=torch.zeros(rows, dtype=torch.int32, device="cuda"), probs=torch.zeros(rows, device="cuda"))
    s = dict(case=c, **_batch(c, g))
    s.update(_cache(c, s["n_pages"], g))
    rows, heads, kvh, hd = s["rows"], c["heads"], c["kv_heads"], c["hd"]
    s["q"] = torch.randn(rows, heads, hd, generator=g, device="cuda") * 1.5
    s["out"] = torch.zeros(rows, heads, hd, device="cuda")
    if c["op"] == "append":
        s["k_new"] = torch.randn(rows, kvh, hd, generator=g, device="cuda") * 2.0
        s["v_new"] = torch.randn(rows, kvh, hd, generator=g, device="cuda")
        for name in ("q_norm", "k_norm"):
            s[name] = 1.0 + 0.2 * torch.randn(hd, generator=g, device="cuda") if c["norm"] else None
    return s


# ---------------------------------------------------------------- the plain forms

def _rms(x, w):
    return x if w is None else x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w


def _turn(x, pos, c):
    """x[rows, heads, hd] rotated to positions pos[rows]; the angles in 64 bits."""
    if c["rope"] == "none":
        return x
    half = c["hd"] // 2
    a = pos.double()[:, None] * torch.exp2(torch.arange(half, device=x.device, dtype=torch.float64) * (-2.0 / c["hd"] * math.log2(c["theta"])))
    cos, sin = torch.cos(a).float()[:, None], torch.sin(a).float()[:, None]
    if c["rope"] == "halves":
        p, q = x[..., :half], x[..., half:]
        return torch.cat([p * cos - q * sin, p * sin + q * cos], -1)
    p, q = x[..., 0::2], x[..., 1::2]
    return torch.stack([p * cos - q * sin, p * sin + q * cos], -1).flatten(-2)


def _where(s):
    """(live, position, page, slot) of every new row."""
    c, n = s["case"], s["rows"]
    counts = (s["row0"][1:] - s["row0"][:-1]).long()
    seq = torch.repeat_interleave(torch.arange(s["n_seq"], device="cuda"), counts, output_size=n)
    ctx = s["ctx"].long()[seq]
    pos = ctx + torch.arange(n, device="cuda") - s["row0"].long()[seq]
    at = (pos // c["page"]).clamp(0, s["pages_ld"] - 1)
    page = s["table"].long()[seq, at]
    return ctx >= 0, pos, page, pos.clamp(min=0) % c["page"]


def _plain_append(s):
    c, page_len = s["case"], s["case"]["page"]
    live, pos, page, slot = _where(s)
    q = _turn(_rms(s["q"], s["q_norm"]), pos, c)
    q = torch.where(live[:, None, None], q, s["out"])
    k = _turn(_rms(s["k_new"], s["k_norm"]), pos, c)
    n_live = int(sum(n for n, x in zip(*_lengths(c)) if x >= 0))
    page, slot = page[:n_live], slot[:n_live]          # the idle slots come last
    outs = [q]
    for name, x in (("k", k), ("v", s["v_new"])):
        x = x[:n_live]
        cache, scale = s[name], s[name + "_scale"]
        if c["kv"] == "f16":
            cache[page, :, slot] = x.clamp(-65504.0, 65504.0).half()
            outs.append(cache)
            continue
        # the scale a page needs: the least power of two with amax <= 448 scale; it only grows, unless the page starts anew
        amax = torch.zeros(s["n_pages"], c["kv_heads"], device="cuda").index_reduce_(0, page, x.abs().amax(-1), "amax")
        first = torch.full((s["n_pages"],), page_len, device="cuda").index_reduce_(0, page, slot, "amin")
        m, e = torch.frexp(amax)
        need = torch.exp2((e - torch.where(m <= 0.875, 9, 8)).float().clamp(min=-120.0))
        old = torch.where((first < page_len)[:, None], torch.where((first == 0)[:, None], 0.0, scale), scale)
        now = torch.where((first < page_len)[:, None], torch.maximum(old, need), scale)
        some = torch.argsort((first < page_len).int(), descending=True, stable=True)[: s["touched"]]
        f = (old[some] / now[some])[:, :, None, None]
        raw = cache.view(torch.uint8)
        moved = (cache[some].float() * f).to(torch.float8_e4m3fn).view(torch.uint8)
        raw[some] = torch.where(f > 0, moved, raw[some])
        scale.copy_(now)
        raw[page, :, slot] = (x / now[page][:, :, None]).to(torch.float8_e4m3fn).view(torch.uint8)
        outs += [cache, scale]
    return outs


def _plain_attn(s):
    c, page_len, kvh, hd = s["case"], s["case"]["page"], s["case"]["kv_heads"], s["case"]["hd"]
    n_seq, n, g = s["n_seq"], s["rows"], c["heads"] // c["kv_heads"]
    most, n_tab = s["most"], -(-s["longest"] // page_len)
    table = s["table"][:, :n_tab].long()

    def gathered(name):
        x = s[name][table].float() if c["kv"] == "f16" else s[name][table].float() * s[name + "_scale"][table][..., None, None]
        return x.transpose(1, 2).reshape(n_seq, kvh, n_tab * page_len, hd)

    live, pos, _, _ = _where(s)
    counts = (s["row0"][1:] - s["row0"][:-1]).long()
    seq = torch.repeat_interleave(torch.arange(n_seq, device="cuda"), counts, output_size=n)
    nth = torch.arange(n, device="cuda") - s["row0"].long()[seq]
    q = torch.zeros(n_seq, most, c["heads"], hd, device="cuda")
    q[seq, nth] = s["q"]
    q = q.view(n_seq, most, kvh, g, hd).transpose(1, 2).reshape(n_seq, kvh, most * g, hd)
    score = torch.matmul(q, gathered("k").transpose(-1, -2)) * (1.0 / math.sqrt(hd))
    token = torch.arange(n_tab * page_len, device="cuda")
    end = (s["ctx"].long()[:, None] + torch.arange(most, device="cuda"))[..., None]        # last token a row may see
    seen = (token <= end) & (s["ctx"] >= 0)[:, None, None]
    if c["window"]:
        seen &= token > end - c["window"]
    seen = seen[:, None, :, None].expand(n_seq, kvh, most, g, token.numel()).reshape(n_seq, kvh, most * g, -1)
    score = torch.where(seen, score, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, gathered("v")) / torch.where(total == 0, 1.0, total)
    return o.view(n_seq, kvh, most, g, hd).transpose(1, 2).reshape(n_seq, most, c["heads"], hd)[seq, nth]


def _plain_sample(s):
    x = torch.where(torch.isnan(s["x"]), -math.inf, s["x"]).double()
    rows, n = x.shape
    t, k, top_p = s["temperature"].double()[:, None], s["top_k"].long()[:, None], s["top_p"].double()[:, None]
    w = torch.exp((x - x.amax(-1, keepdim=True)) / torch.where(t > 0, t, 1.0))
    _, order = torch.sort(x, dim=-1, descending=True, stable=True)
    rank = torch.arange(n, device=x.device)[None]
    ws = w.gather(1, order)
    k = torch.where(t > 0, torch.where(k > 0, k, n), 1)
    ws = torch.where(rank < k, ws, 0.0)
    before = torch.cumsum(ws, -1) - ws
    keep = (rank < k) & ((before < top_p * ws.sum(-1, keepdim=True)) | (top_p >= 1.0) | (rank == 0)) & (ws >= s["min_p"].double()[:, None])
    kept = torch.zeros_like(w).scatter_(1, order, torch.where(keep, ws, 0.0))
    upto = torch.cumsum(kept, -1)
    total = upto[:, -1:]
    i = (upto <= s["u"].double()[:, None] * total).sum(-1, keepdim=True)
    i = torch.minimum(i, torch.where(kept > 0, rank, 0).amax(-1, keepdim=True))
    return [i[:, 0].int(), (kept.gather(1, i) / total)[:, 0].float()]


# ---------------------------------------------------------------- the library's calls

_accel = None


def _plan(s):
    """What a user's program makes once for its cache and its batch buffers."""
    global _accel
    from __graft_entry__ import load_package
    pkg = load_package()
    if _accel is None:
        _accel = pkg.CudaWeightAccel(0)
    c = s["case"]
    plan = s["plan"] = dict(acc=_accel)
    if c["op"] == "sample":
        return plan
    ptr = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
    plan["cache"] = pkg.KvPages(ptr(s["k"]), ptr(s["v"]), s["n_pages"], c["kv_heads"], c["page"], c["hd"],
                                type=pkg.KV_F16 if c["kv"] == "f16" else pkg.KV_E4M3, d_k_scale=ptr(s["k_scale"]), d_v_scale=ptr(s["v_scale"]))
    plan["batch"] = pkg.KvBatch(s["n_seq"], s["rows"], ptr(s["row0"]), ptr(s["ctx"]), ptr(s["table"]), s["pages_ld"])
    if c["op"] == "append":
        rope = {"none": pkg.ROPE_NONE, "halves": pkg.ROPE_HALVES, "adjacent": pkg.ROPE_ADJACENT}[c["rope"]]
        plan["prep"] = pkg.KvPrep(rope=rope, theta=c["theta"], d_q_norm=ptr(s["q_norm"]), d_k_norm=ptr(s["k_norm"]), eps=1e-6)
    else:
        plan["work"] = torch.zeros(_accel.attn_pages_workspace(plan["cache"], plan["batch"], c["heads"]), dtype=torch.uint8, device="cuda")
    return plan


def _own_run(s):
    c, plan = s["case"], s.get("plan") or _plan(s)
    acc, stream = plan["acc"], torch.cuda.current_stream().cuda_stream
    if c["op"] == "sample":
        acc.sample_dev(s["x"].data_ptr(), c["n"], c["n"], c["rows"], s["u"].data_ptr(), s["ids"].data_ptr(), d_probs=s["probs"].data_ptr(),
                       d_temperature=s["temperature"].data_ptr(), d_top_k=s["top_k"].data_ptr(), d_top_p=s["top_p"].data_ptr(),
                       d_min_p=s["min_p"].data_ptr(), stream=stream)
        return [s["ids"], s["probs"]]
    if c["op"] == "attn":
        acc.attn_pages_dev(plan["cache"], plan["batch"], c["heads"], s["q"].data_ptr(), s["out"].data_ptr(), 1.0 / math.sqrt(c["hd"]),
                           plan["work"].data_ptr(), plan["work"].numel(), window=c["window"], stream=stream)
        return s["out"]
    acc.kv_append_dev(plan["cache"], plan["batch"], s["k_new"].data_ptr(), s["v_new"].data_ptr(), plan["prep"], n_heads=c["heads"],
                      d_q=s["q"].data_ptr(), d_q_out=s["out"].data_ptr(), stream=stream)
    return [s["out"], s["k"], s["v"]] if c["kv"] == "f16" else [s["out"], s["k"], s["k_scale"], s["v"], s["v_scale"]]


def run(state):
    if own:
        return _own_run(state)
    return {"append": _plain_append, "attn": _plain_attn, "sample": _plain_sample}[state["case"]["op"]](state)


# ---------------------------------------------------------------- the definitions in 64 bits

def _exact_append(c, s):
    new, ctx = _lengths(c)
    P, hd, half = c["page"], c["hd"], c["hd"] // 2
    freq = torch.tensor([c["theta"] ** (-2.0 * j / hd) for j in range(half)], dtype=torch.float64, device="cuda")
    first = torch.arange(half, device="cuda") * (1 if c["rope"] == "halves" else 2)
    second = first + (half if c["rope"] == "halves" else 1)

    def prepared(x, w, at):
        x = x.double()
        if w is not None:
            x = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + 1e-6) * w.double()
        if c["rope"] == "none":
            return x
        z = torch.polar(torch.ones_like(at[:, None] * freq), at[:, None] * freq)[:, None] * torch.complex(x[..., first], x[..., second])
        y = torch.empty_like(x)
        y[..., first], y[..., second] = z.real, z.imag
        return y

    q = s["out"].double().clone()
    cache = {n: s[n].double() for n in ("k", "v")}
    scale = {n: None if c["kv"] == "f16" else s[n + "_scale"].double().clone() for n in ("k", "v")}
    table, row = s["table"].cpu().tolist(), 0
    for i, (n, x) in enumerate(zip(new, ctx)):
        if x >= 0:
            at = torch.arange(x, x + n, dtype=torch.float64, device="cuda")
            q[row:row + n] = prepared(s["q"][row:row + n], s["q_norm"], at)
            rows = {"k": prepared(s["k_new"][row:row + n], s["k_norm"], at), "v": s["v_new"][row:row + n].double()}
            for j in range(x // P, (x + n - 1) // P + 1):
                lo, hi = max(x, j * P), min(x + n, (j + 1) * P)
                pg, a, b = table[i][j], lo - j * P, hi - j * P
                for name in ("k", "v"):
                    y = rows[name][lo - x:hi - x].transpose(0, 1)
                    if c["kv"] == "f16":
                        cache[name][pg, :, a:b] = y.clamp(-65504, 65504)
                        continue
                    need = torch.exp2(torch.ceil(torch.log2(y.abs().amax((1, 2)) / 448.0)).clamp(min=-120))
                    if a:
                        now = torch.maximum(need, scale[name][pg])
                        cache[name][pg] *= (scale[name][pg] / now)[:, None, None]
                    else:
                        now = need
                    cache[name][pg, :, a:b] = y / now[:, None, None]
                    scale[name][pg] = now
        row += n
    return [q, cache["k"], cache["v"]] if c["kv"] == "f16" else [q, cache["k"], scale["k"], cache["v"], scale["v"]]


def _exact_attn(c, s):
    new, ctx = _lengths(c)
    P, g = c["page"], c["heads"] // c["kv_heads"]
    out, table, row = torch.zeros(s["rows"], c["heads"], c["hd"], dtype=torch.float64, device="cuda"), s["table"].long(), 0
    for i, (n, x) in enumerate(zip(new, ctx)):
        if x >= 0:
            pages = table[i, : -(-(x + n) // P)]
            for h in range(c["kv_heads"]):
                k, v = (s[m][pages, h].double() * (1.0 if s[m + "_scale"] is None else s[m + "_scale"][pages, h].double()[:, None, None])
                        for m in ("k", "v"))
                k, v = k.reshape(-1, c["hd"])[: x + n], v.reshape(-1, c["hd"])[: x + n]
                q = s["q"][row:row + n, h * g:(h + 1) * g].double()
                score = torch.einsum("rgd,td->grt", q, k) / math.sqrt(c["hd"])
                token, last = torch.arange(x + n, device="cuda"), torch.arange(x, x + n, device="cuda")[:, None]
                hidden = (token > last) | (token <= last - (c["window"] or x + n + 1))
                p = torch.softmax(score.masked_fill(hidden, -math.inf), -1)
                out[row:row + n, h * g:(h + 1) * g] = torch.einsum("grt,td->rgd", p, v)
        row += n
    return out


def _exact_sample(c, s):
    x = s["x"].cpu().numpy().astype(np.float64)
    par = {k: s[k].cpu().numpy().astype(np.float64) for k in ("temperature", "top_k", "top_p", "min_p", "u")}
    ids, probs = np.zeros(c["rows"], np.int64), np.zeros(c["rows"])
    for r in range(c["rows"]):
        if par["temperature"][r] <= 0:
            ids[r], probs[r] = int(np.argmax(x[r])), 1.0
            continue
        order = np.argsort(-x[r], kind="stable")
        k = int(par["top_k"][r])
        order = order[:k] if k > 0 else order
        w = np.exp((x[r][order] - x[r][order[0]]) / par["temperature"][r])
        if par["top_p"][r] < 1:
            n = int(np.searchsorted(np.cumsum(w), par["top_p"][r] * w.sum(), side="left")) + 1
            order, w = order[:n], w[:n]
        order, w = order[w >= par["min_p"][r]], w[w >= par["min_p"][r]]
        by = np.argsort(order)
        order, w = order[by], w[by]
        i = min(int(np.searchsorted(np.cumsum(w), par["u"][r] * w.sum(), side="right")), len(w) - 1)
        ids[r], probs[r] = order[i], w[i] / w.sum()
    return [torch.from_numpy(ids).int(), probs]


def exact(case, seed):
    """What `run` returns, from the definitions, in 64 bits: stored values before their last rounding, e4m3 ones in units of their scale."""
    s = prepare(case, seed)
    return {"append": _exact_append, "attn": _exact_attn, "sample": _exact_sample}[case["op"]](dict(case), s)
