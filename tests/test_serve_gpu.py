"""The paged KV cache (append, attention) and sampling on the GPU against their definitions in 64 bits."""
import ctypes as C
import math

import numpy as np
import pytest

import serve_oracle as so

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


def _i32(torch, v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Paged:
    """A cache on the device with its page table, and what a test knows about it."""

    def __init__(self, torch, pkg, kv, n_kv, page, hd, tokens, seed=0, pad=0, spare=2, fill=None):
        """tokens: cached capacity of each sequence; pad: extra elements between pages; fill: byte the buffers start with."""
        self.torch, self.pkg, self.kv, self.n_kv, self.page, self.hd = torch, pkg, kv, n_kv, page, hd
        rng = np.random.RandomState(seed)
        need = [-(-t // page) for t in tokens]
        self.n_pages, self.ld = sum(need) + spare, max(need + [1])
        ids = rng.permutation(self.n_pages)
        self.table = np.full((len(tokens), self.ld), -7, np.int32)     # unused entries are no pages
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = ids[at:at + n]
            at += n
        self.stride = n_kv * page * hd + pad
        el = 2 if kv == pkg.KV_F16 else 1
        n = self.n_pages * self.stride * el
        self.raw = {m: torch.full((n,), 0x78 if fill is None else fill, dtype=torch.uint8, device="cuda") for m in "kv"}
        self.scale = {m: torch.full((self.n_pages, n_kv), 1.0, device="cuda") for m in "kv"}
        self.d_table = torch.from_numpy(self.table).cuda()
        self.desc = pkg.KvPages(self.raw["k"].data_ptr(), self.raw["v"].data_ptr(), self.n_pages, n_kv, page, hd, type=kv,
                                d_k_scale=self.scale["k"].data_ptr(), d_v_scale=self.scale["v"].data_ptr(), page_stride=self.stride if pad else 0)

    def values(self, m):
        """float64 [n_pages, n_kv, page, hd]"""
        raw = self.raw[m].cpu().numpy()
        x = raw.view(np.float16) if self.kv == self.pkg.KV_F16 else raw
        x = x.reshape(self.n_pages, self.stride)[:, :self.n_kv * self.page * self.hd].reshape(self.n_pages, self.n_kv, self.page, self.hd)
        if self.kv == self.pkg.KV_F16:
            return x.astype(np.float64)
        return so.e4m3_value(x) * self.scale[m].cpu().numpy().astype(np.float64)[:, :, None, None]

    def tokens(self, m, s, n):
        """float64 [n, n_kv, hd]: the first n cached tokens of sequence s; unused or bad pages as zeros."""
        v, out = self.values(m), np.zeros((n, self.n_kv, self.hd))
        for t in range(n):
            j = t // self.page
            pg = self.table[s, j] if j < self.ld else -1
            if 0 <= pg < self.n_pages:
                out[t] = v[pg, :, t % self.page]
        return out

    def batch(self, row0, ctx, n_rows=None):
        self.row0, self.ctx = _i32(self.torch, row0), _i32(self.torch, ctx)
        return self.pkg.KvBatch(len(ctx), row0[-1] if n_rows is None else n_rows, self.row0.data_ptr(), self.ctx.data_ptr(),
                                self.d_table.data_ptr(), self.ld)

    def seed_random(self, seed, lengths):
        """The first lengths[s] tokens of every sequence as a user might have written them: finite values, scales any power of two.
        Everything else keeps the bytes it has."""
        rng = np.random.RandomState(seed)
        for m in "kv":
            raw = self.raw[m].cpu().numpy().copy()
            sc = np.exp2(rng.randint(-9, -4, (self.n_pages, self.n_kv))).astype(np.float32)
            for s, n in enumerate(lengths):
                for t in range(n):
                    pg = self.table[s, t // self.page]
                    for h in range(self.n_kv):
                        o = pg * self.stride + (h * self.page + t % self.page) * self.hd
                        x = rng.randn(self.hd)
                        if self.kv == self.pkg.KV_F16:
                            raw.view(np.float16)[o:o + self.hd] = x
                        else:
                            code = rng.randint(0, 127, self.hd) | (rng.randint(0, 2, self.hd) << 7)
                            raw[o:o + self.hd] = np.where((code & 127) > 0x68, code & 0xe7, code)
            self.raw[m].copy_(self.torch.from_numpy(raw))
            self.scale[m].copy_(self.torch.from_numpy(sc))


def work_of(torch, accel, P, b, heads):
    n = accel.attn_pages_workspace(P.desc, b, heads)
    assert n > 0
    return torch.zeros(n, dtype=torch.uint8, device="cuda")


def stream(torch):
    return torch.cuda.current_stream().cuda_stream


# ---------------------------------------------------------------- append

def half_step(kv, pkg, x, s):
    """How far a stored value may be from x: half a step of its type there, and the f32 arithmetic that made it (norm,
    rotation: a dozen roundings of 2^-24 of the largest value of the head)."""
    a = np.abs(x)
    if kv == pkg.KV_F16:
        return np.maximum(a * 2.0 ** -11, 2.0 ** -25)
    return np.maximum(a * 2.0 ** -4, s * 2.0 ** -10)


@pytest.mark.parametrize("hd,page", [(64, 16), (96, 32), (128, 64), (192, 128), (256, 16), (128, 128)])
@pytest.mark.parametrize("kv", [0, 1])
@pytest.mark.parametrize("rope,norm", [(1, True), (2, False), (0, True)])
def test_append_many_sequences(torch, pkg, accel, kv, hd, page, rope, norm):
    """Ragged new rows, an idle slot, an empty sequence, rows of nobody, strided inputs, frequency factors, padded pages."""
    n_kv, heads = 2, 6
    new = [1, 0, 5, 2 * page + 3, 1, 1]
    ctx = [0, 4, page - 2, 3, -1, 2 * page]
    row0 = np.cumsum([0] + new).tolist()
    rows, all_rows = row0[-1], row0[-1] + 2
    P = Paged(torch, pkg, kv, n_kv, page, hd, [c + n if c >= 0 else 0 for c, n in zip(ctx, new)], seed=hd + page, pad=32)
    P.seed_random(5, [max(c, 0) for c in ctx])
    before = {m: P.raw[m].clone() for m in "kv"}
    old = {m: P.values(m) for m in "kv"}
    old_scale = {m: P.scale[m].cpu().numpy().copy() for m in "kv"}
    b = P.batch(row0, ctx, all_rows)
    g = torch.Generator(device="cuda").manual_seed(hd + 7 * rope)
    fused = torch.randn(all_rows, (heads + 2 * n_kv) * hd + 4, generator=g, device="cuda") * 3.0   # q | k | v slices of one buffer
    q, k, v = fused[:, :heads * hd], fused[:, heads * hd:(heads + n_kv) * hd], fused[:, (heads + n_kv) * hd:(heads + 2 * n_kv) * hd]
    qn, kn = (1 + 0.1 * torch.randn(hd, generator=g, device="cuda") for _ in range(2))
    freq = 1 + torch.rand(hd // 2, generator=g, device="cuda") * 7
    out = torch.full((all_rows, heads * hd + 8), 7.0, device="cuda")
    prep = pkg.KvPrep(rope=rope, theta=5e5, eps=1e-5, norm_v=norm, d_freq=freq.data_ptr(), d_q_norm=qn.data_ptr() if norm else 0,
                      d_k_norm=kn.data_ptr() if norm else 0)
    ld = fused.shape[1]
    assert accel.kv_append_dev(P.desc, b, k.data_ptr(), v.data_ptr(), prep, n_heads=heads, d_q=q.data_ptr(), d_q_out=out.data_ptr(),
                               ld_k=ld, ld_v=ld, ld_q=ld, ld_q_out=out.shape[1], stream=stream(torch))
    torch.cuda.synchronize()
    assert accel.device_status() == 0
    got = {m: P.values(m) for m in "kv"}
    gq = out.cpu().numpy().astype(np.float64)
    hq, hk, hv = (t.cpu().numpy() for t in (q, k, v))
    wq, wk = (t.cpu().numpy() if norm else None for t in (qn, kn))
    fr = freq.cpu().numpy()
    touched = {}
    for s, (n, c) in enumerate(zip(new, ctx)):
        for i in range(n):
            r = row0[s] + i
            if c < 0:
                assert (gq[r] == 7.0).all()
                continue
            pos = c + i
            want = so.prepared(hq[r].reshape(heads, hd), wq, pos, rope, 5e5, 1e-5, fr, norm)
            tol = 16 * 2.0 ** -24 * np.abs(want).max()
            assert np.abs(gq[r, :heads * hd].reshape(heads, hd) - want).max() <= tol
            pg, slot = P.table[s, pos // page], pos % page
            wk_ = so.prepared(hk[r].reshape(n_kv, hd), wk, pos, rope, 5e5, 1e-5, fr, norm)
            wv_ = so.prepared(hv[r].reshape(n_kv, hd), None, pos, 0, 1.0, 1e-5, None, norm)
            t = touched.setdefault(pg, dict(first=slot, slots={}))
            t["slots"][slot] = dict(k=wk_, v=wv_)
    assert (gq[:, heads * hd:] == 7.0).all() and (gq[rows:] == 7.0).all()
    for pg, t in touched.items():
        for m in "kv":
            for h in range(n_kv):
                s_now = float(P.scale[m][pg, h])
                if kv == pkg.KV_E4M3:
                    amax = max(np.abs(x[m][h]).max() for x in t["slots"].values())
                    want_s = max(so.scale_for(amax), float(old_scale[m][pg, h]) if t["first"] else 0.0)
                    assert s_now == want_s
                for slot, x in t["slots"].items():
                    w = x[m][h]
                    assert (np.abs(got[m][pg, h, slot] - w) <= half_step(kv, pkg, w, s_now) + 16 * 2.0 ** -24 * np.abs(w).max()).all()
                for slot in range(t["first"]):       # earlier tokens: moved to the new scale, at most half a (subnormal) step lost
                    w = old[m][pg, h, slot]
                    assert (np.abs(got[m][pg, h, slot] - w) <= (s_now * 2.0 ** -10 if kv else 0.0)).all()
    # bytes that no token owns keep their values: other pages whole, the padding between pages, slots behind the last token
    el = 2 if kv == pkg.KV_F16 else 1
    for m in "kv":
        a, z = (x.cpu().numpy().reshape(P.n_pages, P.stride * el) for x in (before[m], P.raw[m]))
        own = n_kv * page * hd * el
        assert (a[:, own:] == z[:, own:]).all()
        for pg in range(P.n_pages):
            if pg not in touched:
                assert (a[pg] == z[pg]).all()
                continue
            # slots behind the last token go with the scale as the earlier ones do: bytes stay unless it grew (NaN codes stay NaN)
            last = max(touched[pg]["slots"]) + 1
            x, y = (u[pg, :own].reshape(n_kv, page, hd * el)[:, last:] for u in (a, z))
            for h in range(n_kv):
                if kv == pkg.KV_F16 or not touched[pg]["first"] or float(P.scale[m][pg, h]) == old_scale[m][pg, h]:
                    assert (x[h] == y[h]).all()
                else:
                    vx, vy = so.e4m3_value(x[h]) * float(old_scale[m][pg, h]), so.e4m3_value(y[h]) * float(P.scale[m][pg, h])
                    assert ((np.abs(vx - vy) <= float(P.scale[m][pg, h]) * 2.0 ** -10) | ((x[h] & 127) == 127)).all()


def test_append_token_by_token_grows_the_scale(torch, pkg, accel):
    """Values that double again and again: every code moves down with the scale and stays within one rounding of each growth."""
    hd, page, n_kv = 64, 16, 1
    P = Paged(torch, pkg, pkg.KV_E4M3, n_kv, page, hd, [40])
    rng = np.random.RandomState(3)
    rows = (rng.randn(40, hd) * np.exp2(rng.randint(-6, 7, 40))[:, None]).astype(np.float32)
    prep = pkg.KvPrep(rope=pkg.ROPE_NONE)
    for t in range(40):
        x = torch.from_numpy(rows[t:t + 1]).cuda()
        b = P.batch([0, 1], [t])
        assert accel.kv_append_dev(P.desc, b, x.data_ptr(), x.data_ptr(), prep, stream=stream(torch))
        torch.cuda.synchronize()
    got, sc = P.tokens("k", 0, 40)[:, 0], P.scale["k"].cpu().numpy()
    for t in range(40):
        j = t // page
        first, last = j * page, min(40, (j + 1) * page)
        s = float(sc[P.table[0, j], 0])
        assert s == so.scale_for(np.abs(rows[first:last]).max())
        # one rounding when it came (2^-4 of the value or 2^-10 of the scale then), and less than one subnormal half step,
        # 2^-10 of the final scale, for all later moves together with the first: 1 + 1/2 + 1/4 + ...
        assert (np.abs(got[t] - rows[t]) <= np.abs(rows[t]) * 2.0 ** -4 + 2 * s * 2.0 ** -10).all()
    assert (P.values("k") == P.values("v")).all()


def test_append_special_values_and_recycled_pages(torch, pkg, accel):
    """Zeros, NaN, infinities; a page that starts anew forgets its old scale."""
    for kv in (pkg.KV_F16, pkg.KV_E4M3):
        P = Paged(torch, pkg, kv, 1, 16, 64, [16])
        P.scale["k"].fill_(64.0)
        P.scale["v"].fill_(64.0)
        z = torch.zeros(1, 64, device="cuda")
        prep = pkg.KvPrep(rope=pkg.ROPE_NONE)
        assert accel.kv_append_dev(P.desc, P.batch([0, 1], [0]), z.data_ptr(), z.data_ptr(), prep, stream=stream(torch))
        torch.cuda.synchronize()
        assert (P.tokens("k", 0, 1) == 0).all()
        if kv == pkg.KV_E4M3:
            assert float(P.scale["k"][P.table[0, 0], 0]) == 2.0 ** -120
        x = torch.randn(1, 64, device="cuda")
        x[0, 3], x[0, 5], x[0, 7] = float("nan"), float("inf"), -float("inf")
        assert accel.kv_append_dev(P.desc, P.batch([0, 1], [1]), x.data_ptr(), z.data_ptr(), prep, stream=stream(torch))
        torch.cuda.synchronize()
        got = P.tokens("k", 0, 2)[1, 0]
        assert np.isfinite(got).all() and got[3] == 0
        most = 65504.0 if kv == pkg.KV_F16 else 3.0e38
        assert abs(got[5] - most) <= most * 2.0 ** -4 and got[7] == -got[5]


def test_append_bad_device_data_is_skipped(torch, pkg, accel):
    """Page ids out of range, positions beyond the table, offsets out of range or descending: the good part is stored, the
    status bit is set, nothing else changes."""
    hd, page = 64, 16
    P = Paged(torch, pkg, pkg.KV_F16, 1, page, hd, [32, 32, 32], fill=0)
    P.table[1, 0] = P.n_pages            # out of range
    P.table[2, 1] = -1
    P.d_table.copy_(torch.from_numpy(P.table))
    prep = pkg.KvPrep(rope=pkg.ROPE_HALVES)
    x = torch.ones(60, hd, device="cuda")
    q = torch.zeros(60, hd, device="cuda")
    for row0, ctx, good in (([0, 3, 6, 26], [30, 0, 0], {0: [30, 31], 1: [], 2: list(range(16))}),
                            ([0, 2, 1 << 30, 5], [0, 16, 0], {0: [0, 1], 1: list(range(16, 32)), 2: []})):
        for m in "kv":
            P.raw[m].zero_()
        b = P.batch(row0, ctx, 60)
        assert accel.kv_append_dev(P.desc, b, x.data_ptr(), x.data_ptr(), prep, n_heads=1, d_q=x.data_ptr(), d_q_out=q.data_ptr(), stream=stream(torch))
        torch.cuda.synchronize()
        assert accel.device_status() & 2
        accel.clear_device_status()
        v = P.values("v")
        want = np.zeros_like(v)
        for s, ts in good.items():
            for t in ts:
                if 0 <= P.table[s, t // page] < P.n_pages:
                    want[P.table[s, t // page], 0, t % page] = 1.0
        assert (v == want).all()


def test_append_bad_offsets_that_no_row_leads_to(torch, pkg, accel):
    """Offsets beyond the rows, below zero, going down: the status bit is set whether or not a row lies in such a sequence, rows go
    to the sequences that attention gives them to, and where offsets go down nothing enters but at its place in a sequence that owns it."""
    hd, page = 64, 16
    prep = pkg.KvPrep(rope=pkg.ROPE_NONE)
    for row0, n_rows, whole in (([0, 4, 9], 4, True), ([-3, 0, 4], 4, True), ([0, 5, 3, 8], 8, False), ([0, 5, 3, 8], 10, False), ([0, 9, 2, 3], 60, False),
                                ([0, 1 << 30], 3, True), ([0, 40, 41, -1], 41, True)):
        for many in (False, True):       # a row to a block, a page to a block
            n_seq = len(row0) - 1
            n = n_rows if not many else max(n_rows, 8 * n_seq + 1)
            if many and n != n_rows and max(row0) > n_rows:
                continue                 # (more rows would change what is out of range)
            P = Paged(torch, pkg, pkg.KV_F16, 1, page, hd, [64] * n_seq, fill=0)
            x = (torch.arange(n, device="cuda").float() + 1)[:, None].expand(n, hd).contiguous()
            b = P.batch(row0, [3] * n_seq, n)
            q = torch.zeros_like(x)
            assert accel.kv_append_dev(P.desc, b, x.data_ptr(), x.data_ptr(), prep, n_heads=1, d_q=x.data_ptr(), d_q_out=q.data_ptr(), stream=stream(torch))
            torch.cuda.synchronize()
            assert accel.device_status() == 2, (row0, n)
            accel.clear_device_status()
            got = np.stack([P.tokens(m, s, 64)[:, 0] for m in "kv" for s in range(n_seq)]).reshape(2, n_seq, 64, hd)
            assert (got[0] == got[1]).all()
            clamp = lambda o: min(max(o, 0), n)  # noqa: E731
            for s in range(n_seq):
                for t in range(64):
                    r = clamp(row0[s]) + t - 3
                    owns = t >= 3 and r < clamp(row0[s + 1])
                    assert (got[0, s, t] == got[0, s, t, 0]).all() and got[0, s, t, 0] in ([r + 1.0] if owns and whole else [0.0, r + 1.0] if owns else [0.0])
            hq = q.cpu().numpy()
            assert (((hq == 0) | (hq == x.cpu().numpy())).all())


def test_bad_device_data_stays_with_the_serving_calls(torch, pkg, accel, orc, synth):
    """What a bad page id sets is there to be read and cleared, and no other call takes it for a failure of its own."""
    w, x = synth.q8_0(71, "status", 64, 512), synth.normal(71, "status.x", 512)
    assert accel.upload_q8_0("serve.status", w, 512, 64) and accel.upload_q8_0("serve.status.head", w, 512, 64)
    P = Paged(torch, pkg, pkg.KV_F16, 1, 16, 64, [32], fill=0)
    P.table[0, 0] = P.n_pages
    P.d_table.copy_(torch.from_numpy(P.table))
    row = torch.ones(1, 64, device="cuda")
    b = P.batch([0, 1], [3])
    out = torch.zeros(1, 64, device="cuda")
    work = work_of(torch, accel, P, b, 1)
    appended = lambda: accel.kv_append_dev(P.desc, b, row.data_ptr(), row.data_ptr(), pkg.KvPrep(rope=pkg.ROPE_NONE), stream=stream(torch))  # noqa: E731
    attended = lambda: accel.attn_pages_dev(P.desc, b, 1, row.data_ptr(), out.data_ptr(), 0.125, work.data_ptr(), work.numel(), stream=stream(torch))  # noqa: E731
    want = orc.qmatmul(x, w, synth.Q8_0, 512, 64)
    try:
        for call in (appended, attended):
            assert call()
            torch.cuda.synchronize()
            for got in (accel.gemv("serve.status", x), accel.gemv_rows("serve.status", x[None], 1)[0], accel.gemv_batch([("serve.status", x)])[0]):
                assert np.linalg.norm(got - want) <= 1e-3 * np.linalg.norm(want)   # (the tolerance of the GEMV tests)
            ids = accel.lm_head_argmax_rows("serve.status.head", x[None], 1)
            assert int(ids[0]) == int(np.argmax(want))
            assert accel.device_status() == 2 and accel.device_status() == 2
            assert accel.clear_device_status() and accel.device_status() == 0
    finally:
        accel.clear_device_status()


# ---------------------------------------------------------------- attention

def check_attention(torch, accel, P, b, row0, ctx, heads, q, out, scale, window, hole=None, strict=1.0):
    """Every row against 64 bits. The bound: a score is a sum of hd products of f32 accuracy, so it is off by at most
    (hd + 8) 2^-24 of the sum of their magnitudes (times `strict` <= 1), a probability by twice that relatively, and the sum over v
    adds as many roundings as it has terms, at most 2^-24 each of the largest magnitude; plus 2^-20 for exp and the joins."""
    hq, ho = q.cpu().numpy().reshape(q.shape[0], heads, P.hd), out.cpu().numpy().reshape(q.shape[0], heads, P.hd)
    cap = P.ld * P.page
    for s, c in enumerate(ctx):
        rows = range(row0[s], row0[s + 1])
        if c < 0:
            assert all((ho[r] == 0).all() for r in rows)
            continue
        n = min(c + len(rows), cap)
        k, v = P.tokens("k", s, n), P.tokens("v", s, n)
        for i, r in enumerate(rows):
            h = None if hole is None else hole[s][:n]
            want = so.attend(hq[r], k, v, c + i, scale, window, h)
            g = heads // P.n_kv
            for hh in range(heads):
                mag = np.abs(k[:, hh // g]) @ np.abs(hq[r, hh].astype(np.float64)) * scale
                d = 2 * (P.hd + 8) * 2.0 ** -24 * (mag.max() if n else 0.0) * strict + 2.0 ** -20
                top = np.abs(v[:, hh // g]).max() if n else 0.0
                err = np.abs(ho[r, hh] - want[hh]).max()
                assert err <= d * top, (s, i, hh, err, d * top)


def run_attention(torch, pkg, accel, kv, n_kv, group, page, hd, new, ctx, window=0, seed=1, pad=0, extra=1, qs=1.0, fill=None, ldpad=0):
    heads = n_kv * group
    row0 = np.cumsum([0] + new).tolist()
    P = Paged(torch, pkg, kv, n_kv, page, hd, [c + n if c >= 0 else 0 for c, n in zip(ctx, new)], seed=seed, pad=pad, fill=fill)
    P.seed_random(seed, [c + n if c >= 0 else 0 for c, n in zip(ctx, new)])
    b = P.batch(row0, ctx, row0[-1] + extra)
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.randn(row0[-1] + extra, heads * hd + ldpad, generator=g, device="cuda") * qs
    out = torch.full((row0[-1] + extra, heads * hd + ldpad), 5.0, device="cuda")
    w = work_of(torch, accel, P, b, heads)
    scale = 1.0 / math.sqrt(hd)
    for _ in range(2):      # twice: the workspace is ready for the next call
        out.fill_(5.0)
        assert accel.attn_pages_dev(P.desc, b, heads, q.data_ptr(), out.data_ptr(), scale, w.data_ptr(), w.numel(), window=window,
                                    ld_q=q.shape[1] if ldpad else 0, ld_out=q.shape[1] if ldpad else 0, stream=stream(torch))
        torch.cuda.synchronize()
        assert accel.device_status() == 0
        assert (out[row0[-1]:] == 5.0).all() and (out[:, heads * hd:] == 5.0).all()
        check_attention(torch, accel, P, b, row0, ctx, heads, q[:, :heads * hd].contiguous(), out[:, :heads * hd].contiguous(), scale, window)
    return P, b, row0, q, out, w


@pytest.mark.parametrize("hd,page", [(64, 16), (64, 128), (96, 32), (128, 64), (128, 16), (192, 128), (256, 16), (256, 64)])
@pytest.mark.parametrize("kv", [0, 1])
def test_attention_single_tokens(torch, pkg, accel, kv, hd, page):
    """One new row a sequence, contexts of every ending, an idle slot, a sequence without rows, garbage (NaN codes) behind the end."""
    ctx = [0, 1, 14, 15, 16, 31, page - 1, page, 2 * page + 1, -1, 5, 300]
    new = [1] * 10 + [0, 1]
    run_attention(torch, pkg, accel, kv, 2, 4, page, hd, new, ctx, fill=0xff)


@pytest.mark.parametrize("group", [1, 2, 3, 5, 7, 8, 9, 16, 17])
@pytest.mark.parametrize("kv", [0, 1])
def test_attention_head_groups(torch, pkg, accel, kv, group):
    run_attention(torch, pkg, accel, kv, 3, group, 32, 64, [1, 2, 1], [100, 33, 0], pad=16, ldpad=4)


@pytest.mark.parametrize("window", [0, 1, 5, 16, 40, 100])
@pytest.mark.parametrize("kv,hd,page,group", [(0, 64, 16, 2), (1, 128, 64, 4), (0, 256, 32, 1), (1, 96, 16, 3)])
def test_attention_several_rows_and_windows(torch, pkg, accel, kv, hd, page, group, window):
    run_attention(torch, pkg, accel, kv, 2, group, page, hd, [5, 1, 33, 8, 2], [0, 70, 3, 200, -1], window=window)


@pytest.mark.parametrize("kv,hd,group,rows", [(1, 128, 4, 150), (0, 64, 8, 70), (1, 256, 2, 40), (0, 96, 1, 300)])
def test_attention_prompt_chunks(torch, pkg, accel, kv, hd, group, rows):
    run_attention(torch, pkg, accel, kv, 1, group, 64, hd, [rows, 1, rows // 3], [0, 64, 129])


def test_attention_long_contexts_split_and_joined(torch, pkg, accel):
    run_attention(torch, pkg, accel, pkg.KV_E4M3, 1, 4, 128, 64, [1, 1], [5000, 17])
    run_attention(torch, pkg, accel, pkg.KV_F16, 2, 1, 16, 64, [3], [3001])


def test_attention_most_sequences(torch, pkg, accel):
    """8192 sequences, the most of a call: their running counts fill 32 KB of the memory that the first copies land in."""
    n, page = 8192, 16
    for kv, hd, group in ((pkg.KV_F16, 64, 2), (pkg.KV_F16, 64, 20), (pkg.KV_F16, 128, 20), (pkg.KV_E4M3, 128, 2), (pkg.KV_E4M3, 128, 20)):
        g = torch.Generator(device="cuda").manual_seed(hd + group)
        table = torch.randperm(n, generator=g, device="cuda").int()[:, None].contiguous()
        ctx = torch.randint(0, page, (n,), generator=g, device="cuda").int()
        row0 = torch.arange(n + 1, device="cuda").int()
        x = [torch.randn(n, 1, page, hd, generator=g, device="cuda") for _ in "kv"]
        k, v = (t.half() if kv == pkg.KV_F16 else t.to(torch.float8_e4m3fn) for t in x)
        one = torch.ones(n, 1, device="cuda")
        P = pkg.KvPages(k.data_ptr(), v.data_ptr(), n, 1, page, hd, type=kv, d_k_scale=one.data_ptr(), d_v_scale=one.data_ptr())
        b = pkg.KvBatch(n, n, row0.data_ptr(), ctx.data_ptr(), table.data_ptr(), 1)
        q = torch.randn(n, group, hd, generator=g, device="cuda")
        out = torch.full_like(q, 5.0)
        w = torch.zeros(accel.attn_pages_workspace(P, b, group), dtype=torch.uint8, device="cuda")
        scale = hd ** -0.5
        assert accel.attn_pages_dev(P, b, group, q.data_ptr(), out.data_ptr(), scale, w.data_ptr(), w.numel(), stream=stream(torch))
        torch.cuda.synchronize()
        assert accel.device_status() == 0
        kk, vv = (t[table[:, 0].long(), 0].double() for t in (k, v))
        s = torch.einsum("ngd,ntd->ngt", q.double(), kk) * scale
        s = s.masked_fill((torch.arange(page, device="cuda")[None] > ctx[:, None])[:, None], -math.inf)
        want = torch.softmax(s, -1) @ vv
        # (the bound of check_attention, with the largest sum of magnitudes of all rows)
        mag = float((torch.einsum("ngd,ntd->ngt", q.double().abs(), kk.abs()) * scale).max())
        assert float((out - want).abs().max()) <= (2 * (hd + 8) * 2.0 ** -24 * mag + 2.0 ** -20) * float(vv.abs().max())


def test_attention_extreme_scores(torch, pkg, accel):
    """Scores of thousands: one token has all the weight; and all scores equal."""
    run_attention(torch, pkg, accel, pkg.KV_E4M3, 1, 4, 16, 64, [1, 2], [90, 200], qs=500.0)
    run_attention(torch, pkg, accel, pkg.KV_F16, 1, 4, 16, 64, [1, 2], [90, 200], qs=0.0)


# (rows of a KV head: few, up to 16, many)
@pytest.mark.parametrize("kv,hd,page,group,new", [(0, 64, 16, 2, 1), (1, 128, 16, 4, 2), (0, 192, 16, 4, 3), (1, 64, 64, 4, 4), (0, 128, 32, 8, 4), (1, 64, 16, 8, 5),
                                                  (1, 128, 64, 4, 9)])
def test_attention_scores_beyond_two_to_the_twenty(torch, pkg, accel, kv, hd, page, group, new):
    """Scores of up to 2^40 whose order f32 tells (one dimension, steps of a sixteenth): the largest has all the weight, so the output
    is that token's value, up to what the two halves leave."""
    n = 6 * page + 5
    P = Paged(torch, pkg, kv, 1, page, hd, [n], seed=hd)
    P.seed_random(new, [n])
    P.scale["k"].fill_(1.0)
    rng = np.random.RandomState(new)
    k = np.zeros((n, hd))
    k[:, 0] = np.array([1.0, 1.125, 1.25, 1.5, 0.5, 0.75])[rng.randint(0, 6, n)]
    best = rng.randint(0, n - new)
    k[best, 0] = 1.75
    codes = {0.5: 0x30, 0.75: 0x34, 1.0: 0x38, 1.125: 0x39, 1.25: 0x3a, 1.5: 0x3c, 1.75: 0x3e, 0.0: 0}
    raw = P.raw["k"].cpu().numpy().copy()
    for t in range(n):
        o = P.table[0, t // page] * P.stride + (t % page) * hd
        if kv == pkg.KV_F16:
            raw.view(np.float16)[o:o + hd] = k[t]
        else:
            raw[o:o + hd] = [codes[x] for x in k[t]]
    P.raw["k"].copy_(torch.from_numpy(raw))
    assert (P.tokens("k", 0, n)[:, 0] == k).all()
    v = P.tokens("v", 0, n)[:, 0]
    b = P.batch([0, new], [n - new])
    out = torch.zeros(new, group * hd, device="cuda")
    w = work_of(torch, accel, P, b, group)
    for power in (19, 20, 22, 23, 24, 25, 26, 27, 28, 30, 40):
        for jitter in (1.0, 1.37, 1.9):
            q = torch.zeros(new, group, hd, device="cuda")
            q[..., 0] = 2.0 ** power * jitter
            assert accel.attn_pages_dev(P.desc, b, group, q.data_ptr(), out.data_ptr(), 1.0, w.data_ptr(), w.numel(), stream=stream(torch))
            torch.cuda.synchronize()
            got = out.cpu().numpy().reshape(new, group, hd).astype(np.float64)
            assert (np.abs(got - v[best]) <= 2.0 ** -20 * np.abs(v[best]).max()).all(), (power, jitter)


def test_attention_scales_of_pages_far_apart(torch, pkg, accel):
    """Pages whose scales differ by 2^30: no page overflows or hides another."""
    P, b, row0, q, out, w = run_attention(torch, pkg, accel, pkg.KV_E4M3, 1, 2, 16, 64, [1], [100])
    for m, lo, hi in (("v", -15, 15), ("k", -20, -3)):
        P.scale[m].copy_(torch.exp2(torch.linspace(lo, hi, P.n_pages, device="cuda").round())[:, None])
    assert accel.attn_pages_dev(P.desc, b, 2, q.data_ptr(), out.data_ptr(), 0.125, w.data_ptr(), w.numel(), stream=stream(torch))
    torch.cuda.synchronize()
    check_attention(torch, accel, P, b, row0, [100], 2, q, out, 0.125, 0)


def check_attention_by_weight(P, s, row0, c, heads, q, out, scale, window):
    """The rows of sequence s against 64 bits, with a bound that goes by what a row sees and how much of it: the terms of check_attention
    times sum p |v| of the row, and what two halves of 11 bits lose of a weight (2^-38 of the largest weight times page scale, at codes of
    up to 448: half a step of the smallest f16, 2^-25, where the largest is 2^14 or more, once for each half of a product)."""
    hq, ho = q.cpu().numpy().reshape(q.shape[0], heads, P.hd), out.cpu().numpy().reshape(q.shape[0], heads, P.hd)
    n, g = c + row0[s + 1] - row0[s], heads // P.n_kv
    k, v = P.tokens("k", s, n), P.tokens("v", s, n)
    vs = P.scale["v"].cpu().numpy().astype(np.float64)[P.table[s, np.arange(n) // P.page]]
    for i, r in enumerate(range(row0[s], row0[s + 1])):
        pos = c + i
        see = np.arange(max(0, pos + 1 - window) if window else 0, pos + 1)
        want = so.attend(hq[r], k, v, pos, scale, window)
        for h in range(heads):
            kk, vv, qq = k[see, h // g], v[see, h // g], hq[r, h].astype(np.float64)
            sc = kk @ qq * scale
            p = np.exp(sc - sc.max())
            p /= p.sum()
            d = 2 * (P.hd + 8) * 2.0 ** -24 * (np.abs(kk) @ np.abs(qq) * scale).max() + 2.0 ** -20
            bound = d * (p @ np.abs(vv)).max() + 2.0 ** -38 * 448 * (p * vs[see, h // g]).max()
            assert np.abs(ho[r, h] - want[h]).max() <= bound, (i, h, np.abs(ho[r, h] - want[h]).max(), bound)


# (up to 8 rows a KV head, up to 16, more: the three forms; tiles of 32 and 64 tokens that hold two or four pages)
@pytest.mark.parametrize("apart", [20, 30, 40, 100])
@pytest.mark.parametrize("hd,page,group", [(64, 16, 1), (64, 32, 1), (96, 16, 1), (128, 16, 1), (64, 16, 2), (64, 32, 2), (96, 16, 2), (128, 16, 2),
                                           (96, 16, 5), (64, 16, 4), (64, 32, 4), (128, 16, 4), (128, 32, 4)])
def test_attention_small_page_next_to_a_large_one(torch, pkg, accel, hd, page, group, apart):
    """Rows that see only the page of small scale of a tile (the large one comes later, or lies before the window) are as exact as
    others: no page that a row does not see has a part in its result."""
    new, c = 8, page - 4
    for window in (0, 4):
        P = Paged(torch, pkg, pkg.KV_E4M3, 1, page, hd, [c + new], seed=hd + page)
        P.seed_random(group, [c + new])
        P.scale["k"].fill_(2.0 ** -20)
        for j in (0, 1):       # window 0: rows 0 to 3 see page 0 only; window 4: row 7 sees page 1 only
            P.scale["v"][P.table[0, j]] = 2.0 ** (0 if (j == 0) == bool(window) else -apart)
        b = P.batch([0, new], [c])
        g = torch.Generator(device="cuda").manual_seed(hd)
        q = torch.randn(new, group * hd, generator=g, device="cuda")
        out = torch.zeros_like(q)
        w = work_of(torch, accel, P, b, group)
        assert accel.attn_pages_dev(P.desc, b, group, q.data_ptr(), out.data_ptr(), 0.125, w.data_ptr(), w.numel(), window=window, stream=stream(torch))
        torch.cuda.synchronize()
        check_attention_by_weight(P, 0, [0, new], c, group, q, out, 0.125, window)


@pytest.mark.parametrize("kv,hd,page,group,new", [(1, 128, 64, 4, 1), (1, 192, 16, 2, 1), (0, 128, 64, 4, 1), (1, 128, 64, 4, 4), (0, 64, 32, 16, 1), (1, 256, 32, 4, 6),
                                                  (1, 128, 64, 4, 8), (0, 64, 64, 8, 6)])
def test_attention_small_weights_of_large_values(torch, pkg, accel, kv, hd, page, group, new):
    """One page has nearly all the weight and tiny values, another some 2^-35 of the weight and the values that make the result."""
    n = 2 * page
    c = n - new
    P = Paged(torch, pkg, kv, 1, page, hd, [n], seed=hd)
    P.seed_random(new, [n])
    if kv == pkg.KV_E4M3:
        for j, ks, vs in ((0, 0.5, 2.0 ** -60), (1, 2.0 ** -20, 1.0)):
            P.scale["k"][P.table[0, j]], P.scale["v"][P.table[0, j]] = ks, vs
        qs = 1.0
    else:
        raw = {m: P.raw[m].view(torch.float16).view(P.n_pages, 1, page, hd) for m in "kv"}
        raw["k"][int(P.table[0, 1])] *= 2.0 ** -12
        raw["v"][int(P.table[0, 0])] *= 2.0 ** -14
        P.scale["v"].fill_(2.0 ** -7)       # (for the bound: the largest values are near 4)
        qs = 12.0 * (128 / hd) ** 0.5
    b = P.batch([0, new], [c])
    g = torch.Generator(device="cuda").manual_seed(hd)
    q = torch.randn(new, group * hd, generator=g, device="cuda") * qs
    out = torch.zeros_like(q)
    w = work_of(torch, accel, P, b, group)
    assert accel.attn_pages_dev(P.desc, b, group, q.data_ptr(), out.data_ptr(), 0.125, w.data_ptr(), w.numel(), stream=stream(torch))
    torch.cuda.synchronize()
    check_attention_by_weight(P, 0, [0, new], c, group, q, out, 0.125, 0)


def test_attention_nan_query_stays_in_its_row(torch, pkg, accel):
    for new in ([1, 1], [3, 20]):
        P, b, row0, q, out, w = run_attention(torch, pkg, accel, pkg.KV_E4M3, 1, 2, 16, 64, new, [40, 50])
        good = out.clone()
        q[1, 0] = float("nan")         # row 1, head 0
        assert accel.attn_pages_dev(P.desc, b, 2, q.data_ptr(), out.data_ptr(), 0.125, w.data_ptr(), w.numel(), stream=stream(torch))
        torch.cuda.synchronize()
        assert torch.isnan(out[1, :64]).all()
        out[1, :64] = good[1, :64]
        assert torch.equal(out, good)


def test_attention_bad_device_data_is_masked(torch, pkg, accel):
    """A bad page id hides its tokens; a length beyond the table ends there; a row that then sees nothing gets zeros."""
    page, hd = 16, 64
    for kv in (pkg.KV_F16, pkg.KV_E4M3):
        P = Paged(torch, pkg, kv, 1, page, hd, [64, 16, 48])
        P.seed_random(3, [64, 16, 48])
        P.table[0, 1], P.table[1, 0] = P.n_pages, -5
        P.d_table.copy_(torch.from_numpy(P.table))
        row0, ctx = [0, 1, 2, 4], [60, 10, 46]
        hole = [np.repeat((P.table[s] < 0) | (P.table[s] >= P.n_pages), page) for s in range(3)]
        b = P.batch(row0, ctx, 6)
        q = torch.randn(6, 2 * hd, device="cuda")
        out = torch.full_like(q, 5.0)
        w = work_of(torch, accel, P, b, 2)
        assert accel.attn_pages_dev(P.desc, b, 2, q.data_ptr(), out.data_ptr(), 0.125, w.data_ptr(), w.numel(), stream=stream(torch))
        torch.cuda.synchronize()
        assert accel.device_status() & 2
        accel.clear_device_status()
        assert (out[1] == 0).all() and (out[4:] == 5.0).all()
        check_attention(torch, accel, P, b, row0, ctx, 2, q, out, 0.125, 0, hole=hole)
        # beyond the table: 64 tokens of capacity, the row claims position 1000
        P.table[0, 1] = P.table[2, 0]
        P.d_table.copy_(torch.from_numpy(P.table))
        b = P.batch([0, 1], [1000], 1)
        assert accel.attn_pages_dev(P.desc, b, 2, q.data_ptr(), out.data_ptr(), 0.125, w.data_ptr(), w.numel(), stream=stream(torch))
        torch.cuda.synchronize()
        assert accel.device_status() & 2
        accel.clear_device_status()
        check_attention(torch, accel, P, b, [0, 1], [1000], 2, q[:1], out[:1], 0.125, 0)


@pytest.mark.parametrize("hd,page", [(64, 16), (128, 32), (64, 64), (128, 128), (128, 16)])
@pytest.mark.parametrize("kv", [0, 1])
@pytest.mark.parametrize("window", [0, 3, 70])
def test_attention_row_blocks(torch, pkg, accel, kv, hd, page, window):
    """More than 16 rows a KV head: blocks of 128 rows, ragged ones, several to a sequence, next to single tokens, an idle slot and a
    sequence without rows; garbage (NaN codes) behind the ends; padded pages and rows that do not start on 16 bytes."""
    run_attention(torch, pkg, accel, kv, 2, 4, page, hd, [33, 1, 70, 0, 9, 4], [0, 130, 61, 20, -1, 300], window=window, fill=0xff,
                  pad=0 if window else 48, ldpad=1 if window == 3 else 4 if window else 0)


@pytest.mark.parametrize("kv,hd", [(0, 128), (1, 128), (1, 64)])
def test_attention_row_blocks_split_and_joined(torch, pkg, accel, kv, hd):
    """Long contexts, so that several blocks share a row block and join; 40 rows of one head are one block, 140 two."""
    run_attention(torch, pkg, accel, kv, 1, 4, 64, hd, [10, 35], [4003, 2500])


def test_attention_row_blocks_extreme_scores_and_scales(torch, pkg, accel):
    for kv in (pkg.KV_E4M3, pkg.KV_F16):
        run_attention(torch, pkg, accel, kv, 1, 8, 16, 128, [5, 6], [90, 200], qs=500.0)
        run_attention(torch, pkg, accel, kv, 1, 8, 16, 128, [5, 6], [90, 200], qs=0.0)
    P, b, row0, q, out, w = run_attention(torch, pkg, accel, pkg.KV_E4M3, 1, 8, 16, 64, [4], [100])
    for m, lo, hi in (("v", -15, 15), ("k", -20, -3)):
        P.scale[m].copy_(torch.exp2(torch.linspace(lo, hi, P.n_pages, device="cuda").round())[:, None])
    for scale in (0.125, -0.125, 0.0):
        assert accel.attn_pages_dev(P.desc, b, 8, q.data_ptr(), out.data_ptr(), scale, w.data_ptr(), w.numel(), stream=stream(torch))
        torch.cuda.synchronize()
        # (a negative scale: the bound counts magnitudes)
        check_attention(torch, accel, P, b, row0, [100], 8, q if scale >= 0 else -q, out, abs(scale), 0)


def test_attention_row_blocks_nan_query_and_bad_pages(torch, pkg, accel):
    P, b, row0, q, out, w = run_attention(torch, pkg, accel, pkg.KV_E4M3, 1, 4, 16, 64, [9, 20], [40, 50])
    good = out.clone()
    q[1, 64] = float("nan")            # row 1, head 1
    assert accel.attn_pages_dev(P.desc, b, 4, q.data_ptr(), out.data_ptr(), 0.125, w.data_ptr(), w.numel(), stream=stream(torch))
    torch.cuda.synchronize()
    assert torch.isnan(out[1, 64:128]).all()
    out[1, 64:128] = good[1, 64:128]
    assert torch.equal(out, good)
    for kv in (pkg.KV_F16, pkg.KV_E4M3):
        P = Paged(torch, pkg, kv, 1, 16, 128, [64, 16, 48], fill=0xff)
        P.seed_random(3, [64, 16, 48])
        P.table[0, 1], P.table[1, 0] = P.n_pages, -5
        P.d_table.copy_(torch.from_numpy(P.table))
        row0, ctx = [0, 6, 11, 22], [58, 3, 37]
        hole = [np.repeat((P.table[s] < 0) | (P.table[s] >= P.n_pages), 16) for s in range(3)]
        q = torch.randn(24, 4 * 128, device="cuda")
        out = torch.full_like(q, 5.0)
        b = P.batch(row0, ctx, 24)
        w = work_of(torch, accel, P, b, 4)
        assert accel.attn_pages_dev(P.desc, b, 4, q.data_ptr(), out.data_ptr(), 0.125, w.data_ptr(), w.numel(), stream=stream(torch))
        torch.cuda.synchronize()
        assert accel.device_status() & 2
        accel.clear_device_status()
        assert (out[6:11] == 0).all() and (out[22:] == 5.0).all()
        check_attention(torch, accel, P, b, row0, ctx, 4, q, out, 0.125, 0, hole=hole)


@pytest.mark.parametrize("new,group", [(1, 4), (3, 4), (3, 5), (9, 4)])
@pytest.mark.parametrize("kv,page,hd", [(0, 16, 64), (1, 32, 128), (1, 16, 256)])
def test_attention_window_looks_at_no_page_before_it(torch, pkg, accel, kv, page, hd, new, group):
    """Pages that ended before the first row's window have been given away: their entries are no pages any more."""
    window, ctx = 20, [150, 83, 4 * page + 19]
    row0 = [0, new, 2 * new, 3 * new]
    P = Paged(torch, pkg, kv, 1, page, hd, [c + new for c in ctx], fill=0xff)
    P.seed_random(3, [c + new for c in ctx])
    b = P.batch(row0, ctx)
    g = torch.Generator(device="cuda").manual_seed(3)
    q = torch.randn(3 * new, group * hd, generator=g, device="cuda")
    out = torch.zeros_like(q)
    w = work_of(torch, accel, P, b, group)
    full = P.table.copy()
    for s, c in enumerate(ctx):
        P.table[s, :(c + 1 - window) // page] = -1
    P.d_table.copy_(torch.from_numpy(P.table))
    assert accel.attn_pages_dev(P.desc, b, group, q.data_ptr(), out.data_ptr(), 0.125, w.data_ptr(), w.numel(), window=window, stream=stream(torch))
    torch.cuda.synchronize()
    assert accel.device_status() == 0
    P.table[:] = full
    check_attention(torch, accel, P, b, row0, ctx, group, q, out, 0.125, window)


def test_attention_graph_serves_changing_lengths(torch, pkg, accel):
    """One captured graph, replayed on a stream of its own with other lengths, rows and pages each time; a workspace that larger and
    smaller calls share."""
    for new_max in (1, 24):
        n_seq, hd, page, heads = 3, 128, 32, 4
        P = Paged(torch, pkg, pkg.KV_E4M3, 1, page, hd, [400] * n_seq)
        P.seed_random(9, [400] * n_seq)
        rows = n_seq * new_max
        q = torch.randn(rows, heads * hd, device="cuda")
        out = torch.zeros_like(q)
        b = P.batch([i * new_max for i in range(n_seq + 1)], [0] * n_seq, rows)
        w = work_of(torch, accel, P, b, heads)
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=st):
                assert accel.attn_pages_dev(P.desc, b, heads, q.data_ptr(), out.data_ptr(), 0.1, w.data_ptr(), w.numel(), stream=st.cuda_stream)
        for ctx, new in (([0, 5, 376], [1, 1, 1]), ([300, -1, 64], [1, 1, new_max]), ([376, 376, 376], [new_max] * 3), ([10, 20, 30], [0, 1, 0])):
            row0 = np.cumsum([0] + new).tolist()
            with torch.cuda.stream(st):
                P.row0.copy_(_i32(torch, row0))
                P.ctx.copy_(_i32(torch, ctx))
                out.fill_(5.0)
                g.replay()
            st.synchronize()
            assert accel.device_status() == 0 and (out[row0[-1]:] == 5.0).all()
            check_attention(torch, accel, P, b, row0, ctx, heads, q, out, 0.1, 0)


def test_attention_offsets_that_go_down(torch, pkg, accel):
    """A sequence whose end lies before its start has no rows; offsets that give rows away twice leave everything as it was."""
    for new in (2, 30):
        P = Paged(torch, pkg, pkg.KV_F16, 1, 16, 64, [64] * 4)
        P.seed_random(3, [64] * 4)
        q = torch.randn(4 * new, 2 * 64, device="cuda")
        out = torch.full_like(q, 5.0)
        call = lambda b, w: accel.attn_pages_dev(P.desc, b, 2, q.data_ptr(), out.data_ptr(), 0.125, w.data_ptr(), w.numel(), stream=stream(torch))  # noqa: E731
        b = P.batch([0, 4 * new, 0, 4 * new, 0], [5, 6, -1, 7], 4 * new)       # sequences 0 and 2 both claim all rows
        w = work_of(torch, accel, P, b, 2)
        assert call(b, w)
        torch.cuda.synchronize()
        assert accel.device_status() & 2 and (out == 5.0).all()
        accel.clear_device_status()
        b = P.batch([0, new, new - 1, 2 * new - 1, 2 * new - 1], [5, 6, 7, 8], 4 * new)   # row new - 1 twice, sequence 1 none: not too many
        assert call(b, w)
        torch.cuda.synchronize()
        assert accel.device_status() & 2 and (out[2 * new - 1:] == 5.0).all()
        accel.clear_device_status()
        check_attention(torch, accel, P, b, [0, new - 1], [5], 2, q, out, 0.125, 0)


def test_prompts_and_single_tokens_in_two_calls(torch, pkg, accel):
    """A batch whose single tokens come first, as one call and as two over the same arrays (the second from the first prompt on): the
    same cache bit by bit, the same queries, and attention that agrees with 64 bits either way."""
    hd, page, n_kv, heads, n = 128, 32, 2, 8, 9
    new, ctx = [1] * n + [70, 40], [5, 33, 0, 64, 31, -1, 100, 95, 7] + [0, 50]
    row0 = np.cumsum([0] + new).tolist()
    for kv in (pkg.KV_F16, pkg.KV_E4M3):
        caches = []
        for split in (False, True):
            P = Paged(torch, pkg, kv, n_kv, page, hd, [c + m if c >= 0 else 0 for c, m in zip(ctx, new)], seed=3, fill=0)
            P.seed_random(4, [max(c, 0) for c in ctx])
            b = P.batch(row0, ctx)
            parts = [b] if not split else [
                pkg.KvBatch(n, n, P.row0.data_ptr(), P.ctx.data_ptr(), P.d_table.data_ptr(), P.ld),
                pkg.KvBatch(2, row0[-1], P.row0.data_ptr() + 4 * n, P.ctx.data_ptr() + 4 * n, P.d_table.data_ptr() + 4 * n * P.ld, P.ld)]
            g = torch.Generator(device="cuda").manual_seed(1)
            q, k, v = (torch.randn(row0[-1], h * hd, generator=g, device="cuda") for h in (heads, n_kv, n_kv))
            out = torch.full_like(q, 5.0)
            w = work_of(torch, accel, P, b, heads)
            for part in parts:
                assert accel.kv_append_dev(P.desc, part, k.data_ptr(), v.data_ptr(), pkg.KvPrep(theta=1e4), n_heads=heads, d_q=q.data_ptr(), d_q_out=q.data_ptr(),
                                           stream=stream(torch))
                assert accel.attn_pages_dev(P.desc, part, heads, q.data_ptr(), out.data_ptr(), 0.09, w.data_ptr(), w.numel(), stream=stream(torch))
            torch.cuda.synchronize()
            assert accel.device_status() == 0
            check_attention(torch, accel, P, b, row0, ctx, heads, q, out, 0.09, 0)
            caches.append([P.raw[m] for m in "kv"] + [P.scale[m] for m in "kv"] + [q])
        assert all(torch.equal(a, z) for a, z in zip(*caches))


def test_attention_on_two_streams_at_once(torch, pkg, accel):
    """Calls that run at the same time, each with its own workspace, give what they give alone, bit by bit."""
    jobs = []
    for i, (new, ctx, group) in enumerate((([1, 1, 1], [900, 17, 3000], 4), ([40, 9], [700, 1500], 4))):
        row0 = np.cumsum([0] + new).tolist()
        P = Paged(torch, pkg, i, 2, 32, 128, [c + n for c, n in zip(ctx, new)], seed=i)
        P.seed_random(i, [c + n for c, n in zip(ctx, new)])
        b = P.batch(row0, ctx)
        q = torch.randn(row0[-1], 2 * group * 128, device="cuda")
        jobs.append((P, b, 2 * group, q, torch.zeros_like(q), work_of(torch, accel, P, b, 2 * group), torch.cuda.Stream()))
    go = lambda P, b, heads, q, out, w, st: accel.attn_pages_dev(P.desc, b, heads, q.data_ptr(), out.data_ptr(), 0.09, w.data_ptr(), w.numel(),  # noqa: E731
                                                                 stream=st.cuda_stream)
    torch.cuda.synchronize()
    alone = []
    for j in jobs:
        assert go(*j)
        torch.cuda.synchronize()
        alone.append(j[4].clone())
        j[4].zero_()
    torch.cuda.synchronize()
    for _ in range(20):
        assert all(go(*j) for j in jobs)
    torch.cuda.synchronize()
    assert accel.device_status() == 0 and all(torch.equal(j[4], a) for j, a in zip(jobs, alone))


@pytest.mark.parametrize("kv,hd,new", [(0, 64, 1), (1, 128, 3), (1, 256, 4), (0, 64, 6), (1, 128, 9)])
def test_attention_largest_and_smallest_scales(torch, pkg, accel, kv, hd, new):
    """A scale near the ends of f32 with queries that make up for it gives what 1 gives: neither overflows on the way."""
    P, b, row0, q, out, w = run_attention(torch, pkg, accel, kv, 1, 4, 32, hd, [new], [90])
    for scale, qs in ((-3.0e38, -1.0e-38 / 3), (3.0e38, 1.0e-36 / 3), (1.0e-38, 1.0e37), (1.0e-39, 5.0e37)):
        x = q * qs
        assert accel.attn_pages_dev(P.desc, b, 4, x.data_ptr(), out.data_ptr(), scale, w.data_ptr(), w.numel(), stream=stream(torch))
        torch.cuda.synchronize()
        want = torch.from_numpy(x.cpu().numpy().astype(np.float64) * float(np.float32(scale)))       # (the scale in the query, then 1)
        check_attention(torch, accel, P, b, row0, [90], 4, want, out, 1.0, 0)


def test_attention_refuses_a_scale_that_is_no_number(torch, pkg, accel):
    P = Paged(torch, pkg, pkg.KV_F16, 1, 16, 64, [64])
    for new in (1, 40):       # (few rows, many rows)
        b = P.batch([0, new], [10])
        q = torch.zeros(new, 64, device="cuda")
        out = torch.full_like(q, 5.0)
        w = work_of(torch, accel, P, b, 1)
        for scale in (float("nan"), float("inf"), -float("inf")):
            with pytest.raises(pkg.StrixCudaError):
                accel.attn_pages_dev(P.desc, b, 1, q.data_ptr(), out.data_ptr(), scale, w.data_ptr(), w.numel(), stream=stream(torch))
        torch.cuda.synchronize()
        assert (out == 5.0).all()


@pytest.mark.parametrize("hd", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("kv", [0, 1])
@pytest.mark.parametrize("group,rows", [(4, 3), (16, 1), (2, 8), (4, 8), (3, 21)])
def test_attention_nine_and_more_rows_of_a_head(torch, pkg, accel, kv, hd, group, rows):
    """Sixteen rows a warp, and from seventeen on several warps to a worker (head sizes 96, 192, 256) or row blocks: every head size, both
    cache types, contexts long enough to be shared between blocks, other sequences beside, strides that are no multiple of four."""
    run_attention(torch, pkg, accel, kv, 2, group, 32, hd, [rows, rows, rows], [700, 45, 16], fill=0xff, ldpad=0 if rows == 8 else 1)
    run_attention(torch, pkg, accel, kv, 1, group, 16 if hd > 128 else 64, hd, [rows, rows], [1200, -1], window=90)


@pytest.mark.parametrize("hd,group,rows", [(64, 1, 64), (128, 4, 64), (128, 4, 3), (128, 8, 2), (128, 2, 5), (96, 4, 64), (192, 2, 40), (256, 3, 64), (64, 16, 1)])
def test_attention_workspace_of_the_most_rows_serves_all(torch, pkg, accel, hd, group, rows):
    """A workspace for a decode batch of `rows` sequences serves the same rows, or fewer, in fewer sequences: others finish, a prompt
    comes."""
    page, n_kv = 32, 2
    lengths = [30 + rows] * rows
    P = Paged(torch, pkg, pkg.KV_E4M3, n_kv, page, hd, lengths)
    P.seed_random(1, lengths)
    w = work_of(torch, accel, P, P.batch(list(range(rows + 1)), [30] * rows), n_kv * group)
    q = torch.randn(rows, n_kv * group * hd, device="cuda")
    shapes = {(1, rows), (1, max(1, rows // 4)), (max(1, rows // 16), rows), (max(1, rows // 5), rows), (rows, rows), (max(1, rows // 2), rows)}
    for n_seq, n_rows in sorted(shapes):
        row0 = [n_rows * i // n_seq for i in range(n_seq + 1)]
        b = P.batch(row0, [30] * n_seq)
        assert accel.attn_pages_workspace(P.desc, b, n_kv * group) <= w.numel()
        out = torch.zeros(n_rows, n_kv * group * hd, device="cuda")
        assert accel.attn_pages_dev(P.desc, b, n_kv * group, q.data_ptr(), out.data_ptr(), 0.125, w.data_ptr(), w.numel(), stream=stream(torch))
        torch.cuda.synchronize()
        assert accel.device_status() == 0
        if n_seq <= 4:
            check_attention(torch, accel, P, b, row0, [30] * n_seq, n_kv * group, q[:n_rows], out, 0.125, 0)


def test_serving_calls_refuse(torch, pkg, accel):
    """Wrong arguments are errors with a message, other shapes are declined; nothing is launched."""
    P = Paged(torch, pkg, pkg.KV_F16, 2, 16, 64, [32])
    x = torch.zeros(4, 512, device="cuda")
    b, p = P.batch([0, 1], [0]), x.data_ptr()
    w = work_of(torch, accel, P, b, 4)
    other = torch.zeros_like(x)
    attn = lambda **k: accel.attn_pages_dev(P.desc, k.get("b", b), k.get("heads", 4), k.get("q", p), k.get("o", other.data_ptr()), 1.0, k.get("w", w.data_ptr()),  # noqa: E731
                                            k.get("n", w.numel()), ld_q=k.get("ld", 0))
    for kw in (dict(q=0), dict(w=0), dict(w=w.data_ptr() + 16), dict(n=w.numel() - 1), dict(ld=255), dict(o=0), dict(o=p)):
        with pytest.raises(pkg.StrixCudaError):
            attn(**kw)
    assert attn(heads=3) is False and attn(heads=0) is False
    for sizes in ((8193, 8193), (1, 0x7fffffff)):
        many = pkg.KvBatch(*sizes, P.row0.data_ptr(), P.ctx.data_ptr(), P.d_table.data_ptr(), P.ld)
        with pytest.raises(pkg.StrixCudaError):
            attn(b=many)
        with pytest.raises(pkg.StrixCudaError):
            accel.attn_pages_workspace(P.desc, many, 4)
    prep = pkg.KvPrep(rope=pkg.ROPE_HALVES)
    app = lambda **k: accel.kv_append_dev(P.desc, b, k.get("k", p), p, k.get("prep", prep), n_heads=k.get("heads", 0), d_q=k.get("q", 0),  # noqa: E731
                                          d_q_out=k.get("o", 0), ld_k=k.get("ld", 0))
    for kw in (dict(k=0), dict(ld=127), dict(heads=4, q=p), dict(prep=pkg.KvPrep(rope=3)), dict(prep=pkg.KvPrep(rope=1, theta=0.0))):
        with pytest.raises(pkg.StrixCudaError):
            app(**kw)
    samp = lambda **k: accel.sample_dev(k.get("x", p), k.get("n", 16), k.get("stride", 16), k.get("rows", 2), k.get("u", p), k.get("ids", p))  # noqa: E731
    for kw in (dict(x=0), dict(u=0), dict(ids=0), dict(n=0), dict(n=pkg.SAMPLE_MAX_N + 1, rows=1), dict(stride=15), dict(rows=1 << 31)):
        with pytest.raises(pkg.StrixCudaError):
            samp(**kw)
    # nothing to do is done
    assert samp(rows=0)
    none = pkg.KvBatch(0, 0, P.row0.data_ptr(), P.ctx.data_ptr(), P.d_table.data_ptr(), P.ld)
    assert attn(b=none) and accel.kv_append_dev(P.desc, none, p, p, prep)
    torch.cuda.synchronize()
    assert accel.device_status() == 0 and (x == 0).all()


# ---------------------------------------------------------------- sampling

def sample(torch, accel, x, u, temperature=None, top_k=None, top_p=None, min_p=None, stride=None):
    rows, n = x.shape
    stride = stride or n
    buf = torch.full((rows, stride), 9.0e9, device="cuda")
    buf[:, :n] = torch.from_numpy(x).cuda()
    f = lambda a, t: None if a is None else torch.tensor(np.asarray(a), dtype=t, device="cuda")  # noqa: E731
    T, K, TP, MP, U = f(temperature, torch.float32), f(top_k, torch.int32), f(top_p, torch.float32), f(min_p, torch.float32), f(u, torch.float32)
    ids = torch.full((rows,), -1, dtype=torch.int32, device="cuda")
    probs = torch.full((rows,), -1.0, device="cuda")
    p = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
    assert accel.sample_dev(buf.data_ptr(), n, stride, rows, p(U), p(ids), d_probs=p(probs), d_temperature=p(T), d_top_k=p(K), d_top_p=p(TP),
                            d_min_p=p(MP), stream=stream(torch))
    torch.cuda.synchronize()
    return ids.cpu().numpy(), probs.cpu().numpy()


def check_sample(x, u, ids, probs, T=None, K=None, TP=None, MP=None):
    """Equal ids; a probability is off by f32 rounding of the exponent (|x - max| / T at most about 60 where it counts) and of
    the weights: 2^-17 is eight times that."""
    at = lambda a, r, d: d if a is None else float(np.float32(a[r]))  # noqa: E731
    for r in range(x.shape[0]):
        i, p = so.draw(x[r], float(np.float32(u[r])), at(T, r, 1.0), int(at(K, r, 0)), at(TP, r, 1.0), at(MP, r, 0.0))
        assert ids[r] == i, (r, ids[r], i)
        assert abs(probs[r] - p) <= p * 2.0 ** -17, (r, probs[r], p)


@pytest.mark.parametrize("n", [1, 2, 3, 31, 33, 1000, 4097, 50001, 151936])
def test_sample_all_parameters(torch, accel, n):
    rng = np.random.RandomState(n)
    rows = 24
    x = (rng.randn(rows, n) * 3).astype(np.float32)
    x[:, rng.randint(0, n, 5)] += 6
    u = rng.rand(rows).astype(np.float32)
    T = rng.choice([0.0, 0.3, 0.7, 1.0, 1.7], rows)
    K = rng.choice([0, 1, 2, 40, 1000, n, n + 5, -3], rows)
    TP = rng.choice([0.0, 0.1, 0.5, 0.9, 0.95, 1.0, 2.0], rows)
    MP = rng.choice([0.0, 0.01, 0.05, 0.5, 1.0, 3.0], rows)
    ids, probs = sample(torch, accel, x, u, T, K, TP, MP, stride=n + 3)
    check_sample(x, u, ids, probs, T, K, TP, MP)
    ids, probs = sample(torch, accel, x, u)
    check_sample(x, u, ids, probs)
    ids, probs = sample(torch, accel, x, u, top_k=K)
    check_sample(x, u, ids, probs, K=K)
    ids, probs = sample(torch, accel, x, u, top_p=TP)
    check_sample(x, u, ids, probs, TP=TP)


@pytest.mark.parametrize("rows,n", [(31, 33000), (67, 20001), (70, 140000), (150, 5000), (300, 1500), (3, 393216), (32, 300000)])
def test_sample_many_rows(torch, accel, rows, n):
    """More rows than run at once, unaligned ones too (odd n), and the longest."""
    rng = np.random.RandomState(rows)
    x = (rng.randn(rows, n) * 2.5).astype(np.float32)
    x[0, ::7] = np.nan
    x[1, [3, n - 1]] = np.inf
    x[2] = np.float32(0.25) * np.round(x[2] * 4)          # ties
    u = rng.rand(rows).astype(np.float32)
    T, K = rng.choice([0.0, 0.5, 1.0, 1.5], rows), rng.choice([0, 0, 50, 3000, n // 2], rows)
    TP, MP = rng.choice([0.5, 0.9, 1.0], rows), rng.choice([0.0, 0.02], rows)
    ids, probs = sample(torch, accel, x, u, T, K, TP, MP)
    check_sample(x, u, ids, probs, T, K, TP, MP)


def test_sample_cuts_among_very_many_tokens(torch, accel):
    """Flat rows, where a top-p cut falls among tens of thousands of tokens of nearly equal weight, most of them beside the border of
    some bin. The drawn token has its place at u: its kept weights, in index order, pass u of the whole there, to within the rounding of
    the sums (2^-20 of the whole: f32 sums of up to 128 weights, whose exponents are off by 2^-21) and two tokens that the border
    may take in or leave out."""
    rng = np.random.RandomState(7)
    for n, spread in ((151936, 0.02), (151936, 0.5), (40001, 0.3), (262147, 1.0)):
        rows = 24
        x = (rng.randn(rows, n) * spread).astype(np.float32)
        x[::2] = np.round(x[::2] * 4096) / 4096
        u, T, TP = rng.rand(rows).astype(np.float32), rng.choice([0.5, 1.0, 3.0], rows), rng.choice([0.3, 0.62, 0.9, 0.99], rows)
        K = rng.choice([0, n // 2], rows)
        ids, probs = sample(torch, accel, x, u, temperature=T, top_p=TP, top_k=K)
        for r in range(rows):
            order = np.argsort(-x[r].astype(np.float64), kind="stable")
            order = order[:K[r]] if K[r] else order
            w = np.exp((x[r][order].astype(np.float64) - x[r].max()) / float(np.float32(T[r])))
            before = np.cumsum(w) - w
            kept = before < float(np.float32(TP[r])) * w.sum()
            full = np.zeros(n)
            full[order[kept]] = w[kept]
            total, border = full.sum(), w[kept][-1]
            eps = 2.0 ** -20 * total + 2 * border
            near = np.zeros(n, bool)
            near[order[max(0, int(kept.sum()) - 2):int(kept.sum()) + 2]] = True
            i, upto = int(ids[r]), np.cumsum(full)
            assert full[i] > 0 or near[i]
            assert upto[i] - full[i] - eps <= float(u[r]) * total <= upto[i] + eps, (r, i, upto[i] / total, u[r])
            weight = np.exp((float(x[r, i]) - x[r].max()) / float(np.float32(T[r])))
            assert abs(probs[r] - weight / total) <= (2.0 ** -17 + 2 * border / total) * weight / total


def test_sample_ties(torch, accel):
    """Logits from a few values only (whole rows of ties): top-k and top-p cut inside the ties, lower indices first."""
    rng = np.random.RandomState(1)
    for n in (7, 500, 9999, 151936):
        rows = 16
        x = rng.randint(0, 3, (rows, n)).astype(np.float32)
        x[3] = 1.0
        x[4] = np.where(np.arange(n) % 2, 0.0, -0.0)         # equal, whatever their signs
        u = rng.rand(rows).astype(np.float32)
        K = rng.randint(1, n + 1, rows)
        # whole numbers of equal weights: the border falls between tokens, not on one
        TP = (rng.randint(0, 8, rows) + 0.37) / 8
        ids, probs = sample(torch, accel, x, u, top_k=K)
        check_sample(x, u, ids, probs, K=K)
        ids, probs = sample(torch, accel, x, u, top_k=K, top_p=TP)
        check_sample(x, u, ids, probs, K=K, TP=TP)


def test_sample_special_logits(torch, accel):
    inf, nan, n = np.inf, np.nan, 3000
    x = np.random.RandomState(2).randn(12, n).astype(np.float32)
    x[0] = -inf
    x[1] = nan
    x[2, ::2] = -inf
    x[3, ::3] = nan
    x[4, [5, 700, 2999]] = inf
    x[5] = -inf
    x[5, 2999] = -3.0e38
    x[6] = 3.0e38
    x[7] = -inf
    x[7, 17] = inf
    x[8] = x[8] * 1e30
    x[9, 0] = nan
    u = np.array([0.3, 0.9, 0.5, 0.1, 0.7, 0.5, 0.99, 0.2, 0.4, 0.6, 0.0, 1.0], np.float32)
    for kw in (dict(), dict(top_k=[40] * 12), dict(top_p=[0.9] * 12), dict(temperature=[0.0] * 12), dict(top_k=[2] * 12, top_p=[0.6] * 12, min_p=[0.3] * 12)):
        ids, probs = sample(torch, accel, x, u, **kw)
        check_sample(x, u, ids, probs, kw.get("temperature"), kw.get("top_k"), kw.get("top_p"), kw.get("min_p"))


def test_sample_greedy_is_argmax(torch, accel):
    x = np.random.RandomState(4).randn(3, 151936).astype(np.float32)
    ids, probs = sample(torch, accel, x, [0.1, 0.5, 0.999], temperature=[0.0, -1.0, float("nan")])
    assert (ids == x.argmax(1)).all() and (probs == 1.0).all()


def test_sample_follows_the_distribution(torch, accel):
    """u on a grid: the counts of the drawn tokens are their probabilities to within one grid step."""
    n, grid = 5, 1000
    row = np.array([0.1, 2.0, -1.0, 1.0, 0.0], np.float32)
    ids, _ = sample(torch, accel, np.tile(row, (grid, 1)), (np.arange(grid) + 0.5) / grid)
    p = np.exp(row.astype(np.float64)) / np.exp(row.astype(np.float64)).sum()
    assert (np.abs(np.bincount(ids, minlength=n) / grid - p) <= 1.0 / grid + 1e-6).all()


@pytest.mark.parametrize("cap", [0.0, 5.0])
def test_decode_step_sample_draws_from_the_logits_of_the_step(torch, pkg, orc, synth, cap):
    """The token and its probability are those of a draw from decode_step's logits; without a configured model there is none."""
    from test_argmax_gpu import build_model
    hidden, qdim, kvdim, ffn, vocab, n_layers = 512, 768, 256, 1536, 3000, 2
    acc = pkg.CudaWeightAccel(0)
    try:
        assert acc.decode_step_sample(np.zeros(hidden, np.float32), 0, 0.5) is None
        build_model(acc, synth, hidden, qdim, kvdim, ffn, vocab, n_layers)
        assert acc.configure_decode(hidden, qdim // 128, ffn, vocab, n_layers, eps=1e-6, act=pkg.ACT_F32, final_softcap=cap)
        for seed, kw in ((1, dict()), (2, dict(temperature=0.7, top_k=40, top_p=0.9)), (3, dict(temperature=0.0)), (4, dict(min_p=0.1, temperature=1.5))):
            h0, u = synth.normal(90 + seed, "h0", hidden), 0.17 * seed
            logits = acc.decode_step(h0, 0)
            tok, prob = acc.decode_step_sample(h0, 0, u, **kw)
            one = lambda k: None if k not in kw else [kw[k]]  # noqa: E731
            check_sample(logits[None], np.array([u], np.float32), [tok], [prob], one("temperature"), one("top_k"), one("top_p"), one("min_p"))
        assert acc.device_status() == 0
    finally:
        acc.close()


def test_a_layer_serves_a_batch_step_by_step(torch, pkg, accel, synth):
    """The operators as a server runs them, over the framework's own projections: q, k and v rows from quantised weights, append,
    attention, output projection, head, draw, the next tokens' rows from the drawn ids: a prompt of uneven lengths, then single
    tokens; against 64-bit attention over the cache that the steps built, and 64-bit draws from the logits."""
    hid, heads, n_kv, hd, vocab, page = 256, 4, 2, 64, 500, 16
    kinds = dict(q=heads * hd, k=n_kv * hd, v=n_kv * hd, head=vocab)
    for name, dim in kinds.items():
        assert accel.upload_q8_0("serve." + name, synth.quant(8, 60, name, dim, hid), hid, dim)
    assert accel.upload_q8_0("serve.o", synth.quant(8, 60, "o", hid, heads * hd), heads * hd, hid)
    rng = np.random.RandomState(5)
    emb = rng.randn(vocab, hid).astype(np.float32)
    for kv in (pkg.KV_E4M3, pkg.KV_F16):
        P = Paged(torch, pkg, kv, n_kv, page, hd, [40, 40, 40], fill=0)
        ctx, toks = [0, 0, 0], [rng.randint(0, vocab, n) for n in (7, 1, 18)]
        prep = pkg.KvPrep(rope=pkg.ROPE_HALVES, theta=1e4)
        w = torch.zeros(accel.attn_pages_workspace(P.desc, P.batch([0, 7, 8, 26], ctx), heads), dtype=torch.uint8, device="cuda")
        for step in range(4):
            row0 = np.cumsum([0] + [len(t) for t in toks]).tolist()
            x = emb[np.concatenate(toks)]
            project = lambda name, a: np.stack([accel.gemv("serve." + name, r) for r in a])  # noqa: E731
            q, k, v = (torch.from_numpy(project(n, x)).cuda() for n in "qkv")
            b = P.batch(row0, ctx)
            need = accel.attn_pages_workspace(P.desc, b, heads)
            if need > w.numel():
                w = torch.zeros(need, dtype=torch.uint8, device="cuda")
            out = torch.zeros(row0[-1], heads * hd, device="cuda")
            assert accel.kv_append_dev(P.desc, b, k.data_ptr(), v.data_ptr(), prep, n_heads=heads, d_q=q.data_ptr(), d_q_out=q.data_ptr(), stream=stream(torch))
            assert accel.attn_pages_dev(P.desc, b, heads, q.data_ptr(), out.data_ptr(), 0.125, w.data_ptr(), w.numel(), stream=stream(torch))
            torch.cuda.synchronize()
            check_attention(torch, accel, P, b, row0, ctx, heads, q, out, 0.125, 0)
            last = out.cpu().numpy()[[e - 1 for e in row0[1:]]]
            logits = project("head", x[[e - 1 for e in row0[1:]]] + project("o", last))
            u = rng.rand(3).astype(np.float32)
            ids, probs = sample(torch, accel, logits, u, temperature=[0.8, 0.0, 1.2], top_k=[50, 0, 0], top_p=[0.95, 1.0, 0.9])
            check_sample(logits, u, ids, probs, [0.8, 0.0, 1.2], [50, 0, 0], [0.95, 1.0, 0.9])
            ctx = [c + len(t) for c, t in zip(ctx, toks)]
            toks = [[int(i)] for i in ids]
        assert accel.device_status() == 0
