"""The 8-bit paged KV cache (fl_kv8_*): plan, append, gather and attention
against a plain model of the rules in include/fl_cuda.h, in 64 bits.

Tables, codes and gathered values have to be equal (every scaling is by a
power of two, so a code has one right value). The attention's bound counts its
roundings row by row (attention_bound)."""
import ctypes as C

import numpy as np
import pytest

import flb200

torch = pytest.importorskip("torch")

PAGE, BLOCK = 64, 16
HALF = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}  # half a step of 1.0


# ------------------------------------------------------------------- refusals
def config(**kw):
    c = dict(layers=1, heads=4, kv_heads=2, head_dim=64, pages=8, max_seqs=4, max_rows=64, max_ctx=256, type=0, dtype=0)
    c.update(kw)
    return flb200.KV8Config(*(c[n] for n, _ in flb200.KV8Config._fields_))


@pytest.mark.parametrize("bad", [dict(layers=0), dict(heads=0), dict(kv_heads=0), dict(kv_heads=3), dict(head_dim=80),
                                 dict(head_dim=256), dict(pages=0), dict(pages=(1 << 24) + 1), dict(max_seqs=0),
                                 dict(max_seqs=65537), dict(max_rows=0), dict(max_ctx=0), dict(type=2), dict(dtype=3),
                                 dict(heads=4098, kv_heads=2)])
def test_create_refuses(lib, bad):
    c = config(**bad)
    assert not lib.fl_kv8_create(C.byref(c), 0)
    assert lib.err().startswith("kv8_create: ")


def test_null_handles_refused(lib):
    assert not lib.fl_kv8_create(None, 0)
    assert lib.fl_kv8_plan(None, 64, 64, 1, 1, None) == -1
    assert lib.fl_kv8_append(None, 0, 64, 64, 1, 64, 64, None) == -1
    assert lib.fl_kv8_attention(None, 0, 64, 64, 1, 64, 64, 1.0, None, 0, None) == -1
    assert lib.fl_kv8_gather(None, 0, 64, 64, 1, None) == -1
    assert lib.fl_kv8_tables(None, None) == -1
    lib.fl_kv8_destroy(None)


def test_binding_refuses(lib):
    for kw in (dict(type="int4"), dict(dtype="float64")):
        with pytest.raises(flb200.FLError):
            flb200.KV8Cache(lib, layers=1, heads=1, kv_heads=1, head_dim=64, pages=1, max_seqs=1, max_rows=1, max_ctx=1,
                            **kw)


# ------------------------------------------------------------ the plain model
class Model:
    """Tables as lists, codes as float64 [page][kv head][64][head_dim]."""

    def __init__(self, kv_heads, hd, pages, max_seqs, max_rows, max_ctx, type):
        self.top = 127.0 if type == "int8" else 448.0
        self.type, self.max_rows = type, max_rows
        self.mp = -(-max_ctx // PAGE)
        self.bt = np.zeros((max_seqs, self.mp), np.int64)
        self.held = np.zeros(max_seqs, np.int64)
        self.stack = list(range(pages - 1, -1, -1))
        self.status = 0
        self.code = {n: np.zeros((pages, kv_heads, PAGE, hd)) for n in "kv"}
        self.scale = {n: np.zeros((pages, kv_heads, PAGE // BLOCK)) for n in "kv"}
        self.slot = np.zeros(max_rows, np.int64)
        self.pos, self.seq = self.slot.copy(), self.slot.copy()

    def plan(self, ctx, new, max_new):
        n = len(ctx)
        drop = [b for b in range(n) if new[b] < 0]
        need = [-(-(ctx[b] + new[b]) // PAGE) if new[b] > 0 else 0 for b in range(n)]
        take = sum(max(0, need[b] - (0 if b in drop else self.held[b])) for b in range(n))
        have = len(self.stack) + sum(self.held[b] for b in drop)
        bad = any(new[b] > 0 and (ctx[b] < 0 or new[b] > max_new or need[b] > self.mp) for b in range(n)) or \
            sum(max(x, 0) for x in new) > self.max_rows
        self.status = -1 if bad else max(0, take - have)
        self.ctx, self.new = list(ctx), [max(x, 0) for x in new]
        if self.status:
            self.new = [0] * n
        else:
            for b in reversed(drop):
                self.stack += [self.bt[b, j] for j in range(self.held[b] - 1, -1, -1)]
                self.held[b] = 0
            for b in range(n):
                while self.held[b] < need[b]:
                    self.bt[b, self.held[b]] = self.stack.pop()
                    self.held[b] += 1
        self.row_start = np.concatenate([[0], np.cumsum(self.new)])
        self.kv_start = np.concatenate([[0], np.cumsum([c + x if x else 0 for c, x in zip(self.ctx, self.new)])])
        r = 0
        for b in range(n):
            for i in range(self.new[b]):
                p = self.ctx[b] + i
                self.pos[r], self.seq[r] = p, b
                self.slot[r] = self.bt[b, p // PAGE] * PAGE + p % PAGE
                r += 1

    def round(self, y):
        y = np.where(np.isnan(y), 0.0, np.clip(y, -self.top, self.top))
        if self.type == "int8":
            return np.rint(y)
        e = np.maximum(np.frexp(y)[1] - 1, -6)
        q = np.ldexp(1.0, e - 3)
        return np.rint(y / q) * q

    def append(self, k, v):
        for n, x in (("k", k), ("v", v)):
            r = 0
            for b, m in enumerate(self.new):
                i = 0
                while i < m:
                    p = self.ctx[b] + i
                    o = p % BLOCK
                    cnt = min(BLOCK - o, m - i)
                    page, blk = self.bt[b, p // PAGE], p % PAGE // BLOCK
                    rows = x[r + i:r + i + cnt].transpose(1, 0, 2)       # [kv head, rows, hd]
                    a = np.where(np.isfinite(rows), np.abs(rows), 0.0).max((1, 2))
                    f, e = np.frexp(a / self.top)
                    s = np.ldexp(1.0, np.maximum(np.where(a > 0, np.where(f == 0.5, e - 1, e), -100), -100))
                    old = self.scale[n][page, :, blk].copy()
                    if o:
                        s = np.maximum(s, old)
                        w = slice(blk * BLOCK, blk * BLOCK + o)
                        with np.errstate(invalid="ignore"):
                            self.code[n][page, :, w] = self.round(self.code[n][page, :, w] * (old / s)[:, None, None])
                    w = slice(blk * BLOCK + o, blk * BLOCK + o + cnt)
                    self.code[n][page, :, w] = self.round(rows / s[:, None, None])
                    self.scale[n][page, :, blk] = s
                    i += cnt
                r += m

    def values(self, n, b):
        """[positions, kv heads, hd] of sequence b, cached and new."""
        total = self.ctx[b] + self.new[b]
        pages = self.bt[b, :-(-total // PAGE)]
        x = self.code[n][pages] * np.repeat(self.scale[n][pages], BLOCK, 2)[..., None]
        return x.transpose(0, 2, 1, 3).reshape(-1, x.shape[1], x.shape[3])[:total]

    def gather(self, n):
        parts = [self.values(n, b) for b in range(len(self.new)) if self.new[b]]
        return np.concatenate(parts) if parts else None

    def attention(self, q, scale, mask=None):
        """(output, bound's ingredients per (row, head)) in float64."""
        T, H, hd = q.shape
        out, mag, smag, keys = np.zeros((T, H, hd)), np.zeros((T, H, hd)), np.zeros((T, H)), np.ones((T, H))
        vmax = np.zeros((T, H))
        r = 0
        for b, m in enumerate(self.new):
            if not m:
                continue
            K, V = self.values("k", b), self.values("v", b)
            g = H // K.shape[1]
            for i in range(m):
                see = np.arange(len(K)) <= self.ctx[b] + i
                if mask is not None:
                    see[self.ctx[b]:] = mask[r, :m] != 0
                for h in range(H):
                    if not see.any():
                        continue
                    k, v = K[see, h // g], V[see, h // g]
                    s = scale * (k @ q[r, h])
                    p = np.exp(s - s.max())
                    p /= p.sum()
                    out[r, h] = p @ v
                    mag[r, h] = p @ np.abs(v)
                    smag[r, h] = abs(scale) * (np.abs(k) @ np.abs(q[r, h])).max()
                    keys[r, h], vmax[r, h] = len(k), np.abs(v).max()
                r += 1
        return out, (mag, smag, keys, vmax)


def attention_bound(dtype, out, parts, hd):
    """Half a step of the output's type (fp16 steps by 2^-24 below 2^-14, so at
    least 2^-25 there: a row that sees one key of a small V has such outputs),
    plus what the terms lose: a score is
    off by 2^-22 of sum |q k| for an f32 query's two halves and one step of 2^-23
    per 16 dimensions summed (tensor-core sums may truncate), three more for the
    factors; its exponential by as much relatively and 2^-22 of its own; a
    probability by half a step of a half (16-bit queries) or 2^-22 (two halves);
    the sums over the keys by 2^-23 per 16 keys and one for each join. Below 2^-21
    of the largest a probability is a subnormal half: 2^-32 absolutely, of V's
    largest (two for its scale's range)."""
    mag, smag, keys, vmax = parts
    ds = smag * ((2.0 ** -22 if dtype == "float32" else 0.0) + (hd / 16 + 3) * 2.0 ** -23)
    rel = 2 * ds + 2.0 ** -21 + (2.0 ** -22 if dtype == "float32" else 2.0 ** -11) + 2 * (keys / 16 + 40) * 2.0 ** -23
    half = np.maximum(HALF[dtype] * np.abs(out), 2.0 ** -25 if dtype == "float16" else 0.0)
    return half + (rel[..., None] * mag + (keys * 2.0 ** -31 * vmax)[..., None]) * (1 + 2.0 ** -6)


# ------------------------------------------------------------------ GPU tests
def dev(a, dtype=torch.int32):
    return torch.tensor(np.asarray(a), dtype=dtype, device="cuda")


class Pair:
    """A cache on the GPU and its model, driven alike."""

    def __init__(self, gpu, heads=4, kv_heads=2, hd=64, pages=64, max_seqs=8, max_rows=512, max_ctx=1024, type="int8",
                 dtype="float32", layers=1):
        self.m = Model(kv_heads, hd, pages, max_seqs, max_rows, max_ctx, type)
        self.c = flb200.KV8Cache(gpu, layers=layers, heads=heads, kv_heads=kv_heads, head_dim=hd, pages=pages,
                                 max_seqs=max_seqs, max_rows=max_rows, max_ctx=max_ctx, type=type, dtype=dtype)
        self.dtype, self.H, self.Hk, self.hd = dtype, heads, kv_heads, hd
        self.t = {n: torch.as_tensor(v, device="cuda") for n, v in self.c.tables().items()}

    def plan(self, ctx, new, max_new=None, check=True):
        mx = max(1, max(new)) if max_new is None else max_new
        self.c.plan(dev(ctx), dev(new), mx, stream=0)
        self.m.plan(ctx, new, mx)
        if check:
            self.check_tables()

    def check_tables(self):
        m, n = self.m, len(self.m.new)
        got = {k: v.cpu().numpy() for k, v in self.t.items()}
        assert got["status"][0] == m.status
        assert got["n_free"][0] == len(m.stack)
        assert np.array_equal(got["free_pages"][:len(m.stack)], m.stack)
        assert np.array_equal(got["held"], m.held)
        for b in range(len(m.held)):
            assert np.array_equal(got["block_table"][b, :m.held[b]], m.bt[b, :m.held[b]])
        assert np.array_equal(got["row_start"][:n + 1], m.row_start)
        assert np.array_equal(got["kv_start"][:n + 1], m.kv_start)
        for k, w in (("slot", m.slot), ("pos", m.pos), ("row_seq", m.seq)):
            assert np.array_equal(got[k], w), k   # behind the last row: as before

    def rows(self, rng, heads, n=None, scale=1.0):
        n = sum(self.m.new) if n is None else n
        x = rng.standard_normal((n, heads, self.hd)) * scale
        return dev(x, torch.float32).to(getattr(torch, self.dtype))

    def append(self, k, v):
        self.c.append(0, k, v, stream=0)
        self.m.append(k.double().cpu().numpy(), v.double().cpu().numpy())

    def check_values(self):
        want = [self.m.gather(n) for n in "kv"]
        n = len(want[0])
        out = [torch.full((n, self.Hk, self.hd), 7.0, dtype=getattr(torch, self.dtype), device="cuda") for _ in "kv"]
        self.c.gather(0, *out, stream=0)
        for o, w in zip(out, want):
            w = torch.tensor(w).to(o.dtype)   # of the type: fp16 overflows alike
            assert torch.equal(o.cpu(), w), f"{(o.cpu() != w).sum()} of {w.numel()} values differ"

    def check_attention(self, q, scale=None, mask=None, out=None):
        scale = self.hd ** -0.5 if scale is None else scale
        got = torch.full_like(q, 9.0).contiguous() if out is None else out
        self.c.attention(0, q, got, scale, None if mask is None else dev(mask, torch.uint8), stream=0)
        T = sum(self.m.new)
        want, parts = self.m.attention(q[:T].double().cpu().numpy(), float(np.float32(scale)), mask)
        err = np.abs(got[:T].double().cpu().numpy() - want)
        tol = attention_bound(self.dtype, want, parts, self.hd)
        assert not np.isnan(err).any() and (err <= tol).all(), f"{(err / np.maximum(tol, 1e-300)).max():.3g} x the bound"
        return got


@pytest.mark.gpu
def test_plan_life_of_a_batch(gpu):
    """Sequences join, grow, idle, roll back, end; pages run out; lengths out of
    range are refused and change nothing."""
    rng = np.random.default_rng(1)
    p = Pair(gpu, pages=20, max_seqs=9, max_rows=300, max_ctx=500)
    n = 9
    pos = np.zeros(n, int)
    for step in range(60):
        new = np.where(rng.random(n) < 0.2, 0, rng.integers(1, 40, n))
        new = np.minimum(new, 512 - pos)
        end = rng.random(n) < 0.15
        new[end] = -1
        if step % 7 == 3:
            new[rng.integers(n)] = 260           # often too many pages or rows
        p.plan(pos.tolist(), new.tolist(), max_new=260)
        if p.m.status == 0:
            pos = np.where(new < 0, 0, pos + np.maximum(new, 0))
            back = rng.random(n) < 0.3           # rejected drafts
            pos = np.where(back, np.maximum(0, pos - rng.integers(0, 9, n)), pos)
    seen = p.m.status
    for ctx, new, mx in (([-1, 0], [1, 1], 4), ([0, 0], [5, 1], 4), ([511, 0], [2, 1], 4), ([0, 0], [200, 200], 200)):
        p.plan(ctx, new, max_new=mx)
        assert p.m.status == -1
    p.plan([0] * n, [-1] * n)
    assert p.m.status == 0 and len(p.m.stack) == 20
    assert seen >= -1


@pytest.mark.gpu
@pytest.mark.parametrize("nseq", [1, 1500, 5000])
def test_plan_sizes(gpu, nseq):
    """More sequences than threads, row counts on both sides of the cluster's."""
    rng = np.random.default_rng(nseq)
    p = Pair(gpu, pages=4 * nseq + 50, max_seqs=nseq, max_rows=max(6000, 3 * nseq), max_ctx=4000, heads=1, kv_heads=1, hd=32)
    ctx = rng.integers(0, 100, nseq)
    p.plan(ctx.tolist(), rng.integers(0, 3, nseq).tolist(), max_new=2)
    new = rng.integers(0, 2, nseq)
    new[nseq // 2] = 3000
    p.plan((ctx + 2).tolist(), new.tolist(), max_new=3000)
    assert p.m.status == 0


@pytest.mark.gpu
@pytest.mark.parametrize("type", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("hd", [32, 64, 96, 128])
def test_append_and_gather(gpu, hd, dtype, type):
    """Prompts, single tokens that grow a block's scale, drafts rolled back, a
    sequence that starts over in recycled pages."""
    rng = np.random.default_rng(hd)
    p = Pair(gpu, heads=3, kv_heads=3, hd=hd, dtype=dtype, type=type)
    pos = np.array([0, 0, 0, 0])
    steps = [[70, 1, 0, 33], [1, 1, 5, 16], [1, 3, 1, 0], [7, 1, 1, 1], [2, 64, 1, 15], [1, 1, -1, 1], [1, 1, 40, 1]]
    for i, new in enumerate(steps):
        pos = np.where(np.array(new) < 0, 0, pos)
        p.plan(pos.tolist(), new)
        scale = 2.0 ** rng.uniform(-3, 3)
        p.append(p.rows(rng, 3, scale=scale), p.rows(rng, 3, scale=scale))
        p.check_values()
        pos = pos + np.maximum(new, 0)
        pos = np.maximum(0, pos - np.where(rng.random(4) < 0.4, rng.integers(0, 5, 4), 0))
    again = p.rows(rng, 3)
    p.append(again, again)
    p.append(again, again)      # the same rows once more: the same codes
    p.check_values()


@pytest.mark.gpu
@pytest.mark.parametrize("type", ["int8", "e4m3"])
def test_append_special_values(gpu, type):
    """Zeros, infinities, NaN, exact borders of the scale, ties, extreme sizes."""
    rng = np.random.default_rng(3)
    p = Pair(gpu, heads=1, kv_heads=1, hd=32, type=type)
    x = rng.standard_normal((128, 1, 32))
    x[0:16] = 0.0
    x[20, 0, 3], x[21, 0, 4], x[22, 0, 5] = np.inf, -np.inf, np.nan
    x[32:48] = np.inf
    top = 127.0 if type == "int8" else 448.0
    x[48:64] = np.linspace(-top, top, 512).reshape(16, 1, 32)
    x[64:80] = np.linspace(-top, top, 512).reshape(16, 1, 32) * (1 + 2.0 ** -23)
    x[80:96] = (np.arange(512).reshape(16, 1, 32) % 254 - 127) / 2.0    # ties
    x[96] *= 1e38
    x[100] *= 1e-30
    x[112:128] *= 1e-38
    p.plan([0], [128])
    k = dev(x, torch.float32)
    p.append(k, -k)
    p.check_values()
    p.plan([128], [3])
    p.append(k[:3], k[96:99])
    p.check_values()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_strided_and_short_rows(gpu, dtype):
    """K, V and Q as slices of one fused buffer at aligned and odd offsets; rows
    behind the planned ones, and planned ones behind the buffer, are left alone."""
    rng = np.random.default_rng(4)
    H, Hk, hd = 4, 2, 64
    for pad, new in ((0, 30), (1, 30), (8, 30), (0, 99), (1, 99)):
        p = Pair(gpu, heads=H, kv_heads=Hk, hd=hd, dtype=dtype)
        p.plan([0, 0], [21, new])
        T = 21 + new
        w = (H + 2 * Hk) * hd + pad
        buf = dev(rng.standard_normal((T + 6) * w + 16), torch.float32).to(getattr(torch, dtype))
        at = lambda off, heads: buf.as_strided((T + 6, heads, hd), (w, hd, 1), off)
        q, k, v = at(pad, H), at(pad + H * hd, Hk), at(pad + (H + Hk) * hd, Hk)
        p.append(k, v)
        p.check_values()
        obuf = torch.full(((T + 6) * w + 16,), 3.0, dtype=buf.dtype, device="cuda")
        out = obuf.as_strided((T + 6, H, hd), (w, hd, 1), pad)
        p.check_attention(q, out=out)
        touched = torch.zeros_like(obuf, dtype=torch.bool)
        touched.as_strided((T, H, hd), (w, hd, 1), pad).fill_(True)
        assert (obuf[~touched] == 3.0).all()
        # a shorter output: its rows only
        ob2 = torch.full((T, H, hd), 3.0, dtype=buf.dtype, device="cuda")
        p.c.attention(0, q[:20], ob2[:20], stream=0)
        assert (ob2[20:] == 3.0).all() and torch.equal(ob2[:20], out[:20])


FORMS = [
    # heads, kv_heads, hd, cached lengths, new rows
    (4, 4, 96, [129], [1]),
    (8, 2, 64, [0, 1, 15, 16, 17, 63, 64, 65], [1] * 8),
    (5, 1, 32, [0, 100, 300, 7], [1, 0, 5, 9]),
    (8, 1, 128, [1000, 30, 0], [1, 7, 4]),
    (40, 10, 128, [200, 77], [3, 1]),
    (3, 3, 64, [500, 0], [40, 33]),
    (4, 1, 128, [130, 0, 1], [70, 129, 33]),
    (14, 2, 96, [0, 61], [61, 20]),
    (6, 2, 32, [900], [150]),
    (2, 2, 64, [500, 0], [200, 193]),
    (8, 1, 96, [33, 70], [24, 33]),
]


@pytest.mark.gpu
@pytest.mark.parametrize("type", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("form", range(len(FORMS)))
def test_attention(gpu, form, dtype, type):
    H, Hk, hd, ctx, new = FORMS[form]
    rng = np.random.default_rng(form)
    p = Pair(gpu, heads=H, kv_heads=Hk, hd=hd, dtype=dtype, type=type, max_rows=1200, max_ctx=1200, pages=100)
    p.plan([0] * len(ctx), ctx)
    if sum(ctx):
        p.append(p.rows(rng, Hk, scale=2.0), p.rows(rng, Hk))
    p.plan(ctx, new)
    p.append(p.rows(rng, Hk, scale=2.0), p.rows(rng, Hk))
    q = p.rows(rng, H)
    p.check_attention(q)
    p.check_attention(q * 50, scale=0.02)
    p.check_attention(q, scale=-0.1)


@pytest.mark.gpu
@pytest.mark.parametrize("type", ["int8", "e4m3"])
@pytest.mark.parametrize("new,group", [([5, 7, 1], 1), ([33, 20, 65], 4), ([3, 40, 1], 2)])
def test_attention_masks(gpu, new, group, type):
    """Random masks, rows that see no new row, rows that see nothing at all (an
    empty cache): zeros."""
    rng = np.random.default_rng(5)
    for dtype in ("float32", "float16"):
        p = Pair(gpu, heads=2 * group, kv_heads=2, hd=64, dtype=dtype, type=type)
        ctx = [90, 0, 64]
        p.plan([0] * 3, ctx)
        p.append(p.rows(rng, 2), p.rows(rng, 2))
        p.plan(ctx, new)
        p.append(p.rows(rng, 2), p.rows(rng, 2))
        T, M = sum(new), max(new) + 3
        mask = (rng.random((T, M)) < 0.4).astype(np.uint8)
        mask[0] = 0
        mask[new[0]] = 0                # first row of the sequence without cached positions
        q = p.rows(rng, 2 * group)
        out = p.check_attention(q, mask=mask)
        assert (out[new[0]] == 0).all()


@pytest.mark.gpu
def test_attention_split_and_long(gpu):
    """Lengths that no CTA takes alone, next to short ones; both kernels."""
    rng = np.random.default_rng(6)
    for new in ([1, 1, 2], [1, 100, 60]):
        p = Pair(gpu, heads=4, kv_heads=1, hd=128, dtype="bfloat16", pages=600, max_seqs=3, max_rows=24000, max_ctx=21000)
        ctx = [20000, 7, 3000]
        p.plan([0] * 3, ctx, check=False)
        p.append(p.rows(rng, 1, scale=3.0), p.rows(rng, 1))
        p.plan(ctx, new, check=False)
        p.append(p.rows(rng, 1, scale=3.0), p.rows(rng, 1))
        q = p.rows(rng, 4)
        a = p.check_attention(q)
        b = p.check_attention(q)
        assert torch.equal(a, b)      # joins are in a fixed order


@pytest.mark.gpu
@pytest.mark.parametrize("type", ["int8", "e4m3"])
def test_positions_behind_the_sequence_do_not_matter(gpu, type):
    """Recycled pages full of the largest codes behind the last position, and
    rolled-back rows with other scales."""
    rng = np.random.default_rng(7)
    for nb in (1, 60, 110):
        p = Pair(gpu, heads=2, kv_heads=1, hd=64, dtype="float16", type=type, pages=6, max_seqs=2, max_ctx=384)
        p.plan([0], [384])
        big = torch.full((384, 1, 64), 60000.0, dtype=torch.float16, device="cuda")
        p.append(big, big)
        p.plan([0], [-1])
        p.plan([0], [75])
        p.append(p.rows(rng, 1), p.rows(rng, 1))
        p.plan([75], [nb])
        p.append(p.rows(rng, 1), p.rows(rng, 1))
        p.check_attention(p.rows(rng, 2))
        # V's scales far apart
        p.plan([10], [nb])
        p.append(p.rows(rng, 1), p.rows(rng, 1, scale=2.0 ** -12))
        p.check_attention(p.rows(rng, 2))


@pytest.mark.gpu
def test_rows_stand_alone(gpu):
    """A NaN in one query row, or an infinity, stays in that row and head."""
    rng = np.random.default_rng(8)
    for new in (3, 80, 100):
        p = Pair(gpu, heads=2, kv_heads=1, hd=64)
        p.plan([0], [50])
        p.append(p.rows(rng, 1), p.rows(rng, 1))
        p.plan([50], [new])
        p.append(p.rows(rng, 1), p.rows(rng, 1))
        q = p.rows(rng, 2)
        good = p.check_attention(q)
        for bad in (float("nan"), float("inf")):
            q2 = q.clone()
            q2[1, 1, 5] = bad
            out = torch.empty_like(q2)
            p.c.attention(0, q2, out, stream=0)
            keep = torch.ones((new, 2), dtype=torch.bool, device="cuda")
            keep[1, 1] = False
            assert torch.equal(out[keep], good[keep])
            assert torch.isnan(out[1, 1]).all()


@pytest.mark.gpu
def test_refused_plan_has_no_rows(gpu):
    rng = np.random.default_rng(9)
    p = Pair(gpu, pages=4, max_ctx=512)
    p.plan([0, 0], [64, 64])
    p.append(p.rows(rng, 2), p.rows(rng, 2))
    p.plan([64, 64], [100, 100], max_new=100)
    assert p.m.status == 2
    k = dev(rng.standard_normal((200, 2, 64)), torch.float32)
    q = dev(rng.standard_normal((200, 4, 64)), torch.float32)
    out = torch.full_like(q, 5.0)
    p.c.append(0, k, k, stream=0)
    p.c.attention(0, q, out, stream=0)
    p.c.gather(0, k.clone(), k.clone(), stream=0)
    assert (out == 5.0).all()
    p.plan([64, 64], [1, 0])
    p.append(p.rows(rng, 2), p.rows(rng, 2))
    p.check_values()


@pytest.mark.gpu
def test_gpu_refusals(gpu):
    p = Pair(gpu, layers=2)
    k = torch.zeros((1, 2, 64), device="cuda")
    q = torch.zeros((1, 4, 64), device="cuda")
    with pytest.raises(flb200.FLError, match="no plan"):
        p.c.append(0, k, k)
    p.plan([0], [1])
    for call in (lambda: p.c.append(2, k, k), lambda: p.c.append(-1, k, k), lambda: p.c.append(0, k.half(), k),
                 lambda: p.c.append(0, k.cpu(), k), lambda: p.c.append(0, k[:, :1], k[:, :1]),
                 lambda: p.c.append(0, k.expand(3, 2, 64), k), lambda: p.c.attention(0, q, q[:0]),
                 lambda: p.c.attention(0, q, q.clone(), float("nan")), lambda: p.c.attention(0, q, q.clone(), float("inf")),
                 lambda: p.c.attention(0, k, k), lambda: p.c.plan(dev([0] * 9), dev([1] * 9), 1),
                 lambda: p.c.plan(dev([0]), dev([1]), 0), lambda: p.c.plan(dev([0, 0]), dev([1]), 1),
                 lambda: p.c.attention(0, q, q.clone(), mask=torch.zeros((1, 1), device="cuda"))):
        with pytest.raises(flb200.FLError):
            call()
    p.plan([0], [3], max_new=4)
    q3 = torch.zeros((3, 4, 64), device="cuda")
    with pytest.raises(flb200.FLError, match="shorter than max_new"):
        p.c.attention(0, q3, q3.clone(), mask=torch.ones((3, 3), dtype=torch.uint8, device="cuda"))
    host = np.zeros(4096, np.float32)
    for rc in (gpu.fl_kv8_append(p.c.h, 0, flb200.ptr(host), flb200.ptr(host), 1, 128, 128, None),
               gpu.fl_kv8_attention(p.c.h, 0, q.data_ptr(), flb200.ptr(host), 1, 256, 256, 1.0, None, 0, None),
               gpu.fl_kv8_gather(p.c.h, 0, flb200.ptr(host), flb200.ptr(host), 1, None),
               gpu.fl_kv8_plan(p.c.h, flb200.ptr(host), flb200.ptr(host), 1, 1, None)):
        assert rc == -1 and "not device memory" in gpu.err()
    p.c.append(1, k[:0], k[:0])     # nothing is nothing
    p.c.attention(1, q[:0], q[:0])


@pytest.mark.gpu
def test_streams_graphs_and_two_caches(gpu):
    """A step captured on a stream and replayed as the lengths on the device
    grow; another cache used between the replays on another stream."""
    rng = np.random.default_rng(10)
    p, o = (Pair(gpu, heads=4, kv_heads=2, hd=64, dtype="float16") for _ in range(2))
    for x in (p, o):
        x.plan([0, 0], [30, 64])
        x.append(x.rows(rng, 2), x.rows(rng, 2))
    ctx, new = dev([30, 64]), dev([2, 1])
    k, v, q = p.rows(rng, 2, 3), p.rows(rng, 2, 3), p.rows(rng, 4, 3)
    out = torch.zeros_like(q)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())

    def step():
        p.c.plan(ctx, new, 2, stream=s.cuda_stream)
        p.c.append(0, k, v, stream=s.cuda_stream)
        p.c.attention(0, q, out, stream=s.cuda_stream)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        with torch.cuda.graph(g, stream=s):
            step()
    pos = [30, 64]
    for i in range(5):
        for t in (k, v, q):
            t.copy_(p.rows(rng, t.shape[1], 3))
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            g.replay()
        o.plan([30 + i, 64 + i], [1, 1])
        o.append(o.rows(rng, 2), o.rows(rng, 2))
        o.check_attention(o.rows(rng, 4))
        torch.cuda.synchronize()
        p.m.plan(pos, [2, 1], 2)
        p.m.append(k.double().cpu().numpy(), v.double().cpu().numpy())
        p.check_tables()
        p.check_values()
        want, parts = p.m.attention(q.double().cpu().numpy(), 0.125)
        assert (np.abs(out.double().cpu().numpy() - want) <= attention_bound("float16", want, parts, 64)).all()
        pos = [pos[0] + 2, pos[1] + 1]
        ctx += new


@pytest.mark.gpu
def test_library_stream(gpu):
    """stream None: the library's own, drained by fl_cuda_sync."""
    rng = np.random.default_rng(11)
    p = Pair(gpu)
    ctx, new = dev([0]), dev([40])
    k, q = dev(rng.standard_normal((40, 2, 64)), torch.float32), dev(rng.standard_normal((40, 4, 64)), torch.float32)
    out = torch.zeros_like(q)
    torch.cuda.synchronize()
    p.c.plan(ctx, new, 40)
    p.c.append(0, k, k)
    p.c.attention(0, q, out)
    gpu.check(gpu.fl_cuda_sync(), "sync")
    p.m.plan([0], [40], 40)
    p.m.append(k.double().cpu().numpy(), k.double().cpu().numpy())
    want, parts = p.m.attention(q.double().cpu().numpy(), 0.125)
    assert (np.abs(out.double().cpu().numpy() - want) <= attention_bound("float32", want, parts, 64)).all()


@pytest.mark.gpu
def test_serving_steps(gpu, orc):
    """The operators as a scheduler uses them, over two layers: prompts join a
    running batch, tokens are projected (fl_cuda_matmul_i8), appended, attended,
    projected to logits and sampled; drafts roll back; a sequence ends and
    another takes its pages. Tables, cache and attention equal the model's at
    every step, and every token the sampling rule's on the GPU's logits."""
    from test_sample_rows import expect
    rng = np.random.default_rng(12)
    H, Hk, hd, V, d, layers = 4, 2, 64, 1000, 256, 2
    kw = dict(heads=H, kv_heads=Hk, hd=hd, pages=24, max_seqs=4, max_rows=300, max_ctx=400)
    p = Pair(gpu, layers=layers, **kw)
    second = Model(Hk, hd, 24, 4, 300, 400, "int8")   # the other layer's codes
    w, sc = gpu.synth_q4_0_i8(7, 900, V, d)
    lm = flb200.block_tensor(w, sc)
    gpu.check(gpu.fl_cuda_upload_tensor(C.byref(lm)), "upload")
    pos = np.zeros(4, int)
    plans = [[37, 0, 64, 0], [1, 100, 1, 0], [5, 1, 1, 20], [1, 1, -1, 1], [1, 7, 33, 1], [1, 1, 1, 1]]
    for step, new in enumerate(plans):
        pos = np.where(np.array(new) < 0, 0, pos)
        p.plan(pos.tolist(), new)
        second.plan(pos.tolist(), new, max(1, max(new)))
        assert p.m.status == 0
        T = sum(p.m.new)
        x = p.rows(rng, H, T)
        for layer, m in ((0, p.m), (1, second)):
            k, v = p.rows(rng, Hk, T, 2.0), p.rows(rng, Hk, T)
            p.c.append(layer, k, v, stream=0)
            m.append(k.double().cpu().numpy(), v.double().cpu().numpy())
            out = torch.empty_like(x)
            p.c.attention(layer, x, out, stream=0)
            want, parts = m.attention(x.double().cpu().numpy(), hd ** -0.5)
            assert (np.abs(out.double().cpu().numpy() - want) <= attention_bound("float32", want, parts, hd)).all()
            x = out
        last = p.t["row_start"][1:5].long()[torch.tensor(np.array(p.m.new) > 0, device="cuda")] - 1
        rows = x[last].reshape(len(last), d).contiguous() * 8
        logits = torch.empty((len(last), V), device="cuda")
        gpu.check(gpu.fl_cuda_matmul_i8(rows.data_ptr(), C.byref(lm), logits.data_ptr(), len(last), V, d, C.c_void_p(1)),
                  "matmul")
        u = dev(rng.random(len(last)), torch.float32)
        tok = torch.empty(len(last), dtype=torch.int32, device="cuda")
        tp = torch.full((len(last),), 0.9, device="cuda")
        flb200.sample(gpu, logits, u, tok, top_p=tp, stream=0)
        l, hu = logits.cpu().numpy(), u.cpu().numpy()
        for r in range(len(last)):
            assert int(tok[r]) == expect(orc, l[r], np.float32(1), 0, np.float32(0.9), np.float32(0), hu[r])
        pos = pos + np.maximum(new, 0)
        pos[1] = max(0, pos[1] - step % 3)          # rejected drafts of one sequence


def cold_attention():
    """The first launches of a process: kernels still without their instructions
    in the caches, so that the warps of a CTA run far apart. (For a child process.)"""
    lib = flb200.Lib()
    lib.check(lib.fl_cuda_init(0), "init")
    rng = np.random.default_rng(12)
    p = Pair(lib, pages=24, max_seqs=4, max_rows=300, max_ctx=400)
    for ctx, new in (([0] * 4, [37, 0, 64, 0]), ([37, 0, 64, 0], [1, 100, 1, 0])):
        p.plan(ctx, new)
        p.append(p.rows(rng, 2, scale=2.0), p.rows(rng, 2))
        p.check_attention(p.rows(rng, 4))
    lib.check(lib.fl_cuda_sync(), "sync")


@pytest.mark.gpu
def test_first_launches_of_a_process(gpu):
    import os
    import subprocess
    import sys
    here = os.path.dirname(os.path.abspath(__file__))
    code = f"import sys; sys.path[:0] = {[here, os.path.dirname(flb200.LIB_PATH)]!r}; import test_kv8; test_kv8.cold_attention()"
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


# ------------------------------------------------------- waits that run out
def long_rows(gpu, rng, dtype="bfloat16", ctx=3000, new=300):
    """One sequence whose tiles several CTAs of the kernel for many rows share."""
    p = Pair(gpu, heads=2, kv_heads=1, hd=64, dtype=dtype, pages=80, max_seqs=1, max_rows=4000, max_ctx=4000)
    p.plan([0], [ctx], check=False)
    p.append(p.rows(rng, 1), p.rows(rng, 1))
    p.plan([ctx], [new], check=False)
    p.append(p.rows(rng, 1), p.rows(rng, 1))
    return p, p.rows(rng, 2)


def give_up(gpu, p, q, cta, at):
    out = torch.full_like(q, 9.0)
    rc = gpu.fl_kv8_wait_timeout_check(p.c.h, 0, q.data_ptr(), out.data_ptr(), q.shape[0], q.stride(0), q.stride(0),
                                       p.hd ** -0.5, cta, at, None)
    assert rc == 0, gpu.err()
    return out


def test_timeout_check_refuses(lib):
    for cta, at in ((-1, 1), (0, 0)):
        assert lib.fl_kv8_wait_timeout_check(None, 0, 64, 64, 1, 64, 64, 1.0, cta, at, None) == -1
        assert "out of range" in lib.err()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_a_wait_that_runs_out_is_reported(gpu, dtype):
    """A CTA that stops at any of its groups of products (before the first, between
    the two tiles, with products of one tile under way) ends, reports, and
    leaves the device usable."""
    rng = np.random.default_rng(13)
    other, oq = long_rows(gpu, rng, dtype)
    for at in range(1, 10):
        p, q = long_rows(gpu, rng, dtype)
        torch.cuda.synchronize()
        give_up(gpu, p, q, at % 3, at)
        assert gpu.fl_cuda_sync() == -5, at
        assert gpu.fl_cuda_sync() == 0
        other.check_attention(oq)
        torch.cuda.synchronize()
    assert gpu.fl_cuda_sync() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_a_cache_is_usable_after_a_wait_that_ran_out(gpu, dtype):
    """Tiles that several CTAs share, of which one gave up: they are left unwritten,
    whoever arrives last; the next call on the cache joins them as ever."""
    rng = np.random.default_rng(14)
    p, q = long_rows(gpu, rng, dtype)
    right = p.check_attention(q)
    for cta, at in ((0, 1), (3, 5), (7, 2), (8, 1), (11, 20), (25, 3), (17, 9)):
        torch.cuda.synchronize()
        out = give_up(gpu, p, q, cta, at)
        assert gpu.fl_cuda_sync() == -5, cta
        same = (out == right).flatten(1).all(1)
        unwritten = (out == 9.0).flatten(1).all(1)
        assert (same | unwritten).all() and unwritten.any(), cta
        for _ in range(2):
            q2 = p.rows(rng, 2)
            p.check_attention(q2)
        assert torch.equal(p.check_attention(q), right)


@pytest.mark.gpu
def test_masks_in_host_memory_and_misaligned_lengths_are_refused(gpu):
    p = Pair(gpu)
    p.plan([0], [2])
    q = torch.zeros((2, 4, 64), device="cuda")
    host = np.ones((2, 2), np.uint8)
    assert gpu.fl_kv8_attention(p.c.h, 0, q.data_ptr(), q.data_ptr(), 2, 256, 256, 1.0, flb200.ptr(host), 2, None) == -1
    assert gpu.err() == "kv8_attention: mask is not device memory"
    n = torch.zeros(8, dtype=torch.int32, device="cuda")
    for a, b in ((1, 0), (0, 2)):
        assert gpu.fl_kv8_plan(p.c.h, n.data_ptr() + a, n.data_ptr() + b, 1, 1, None) == -1
        assert "not aligned" in gpu.err()
    assert gpu.fl_cuda_sync() == 0


# ------------------------------------- plans replayed from a graph, calls made eagerly
def replayed_plan(p, ctx, new, max_new, first, rng):
    """A plan for up to max_new rows in a graph; behind its capture a small step is
    planned by a call, then the graph is replayed with the lengths (ctx, new)."""
    c, n = dev(ctx), dev(new)
    s = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=s):
        p.c.plan(c, n, max_new, stream=s.cuda_stream)
    p.plan([0] * len(ctx), ctx)
    p.append(p.rows(rng, p.Hk), p.rows(rng, p.Hk))
    p.plan(ctx, first)
    torch.cuda.synchronize()
    g.replay()
    torch.cuda.synchronize()
    p.m.plan(ctx, new, max_new)
    p.check_tables()
    p.append(p.rows(rng, p.Hk), p.rows(rng, p.Hk))
    return g


@pytest.mark.gpu
@pytest.mark.parametrize("new", [[20, 3], [150, 3]])
def test_masks_narrower_than_a_replayed_plan(gpu, new):
    """New rows behind the mask's columns are not seen, nor read: the call's own
    bound on new rows was that of the step planned by a call."""
    rng = np.random.default_rng(15)
    p = Pair(gpu, heads=2, kv_heads=2, hd=64)
    g = replayed_plan(p, [40, 64], new, 200, [1, 1], rng)
    T = sum(new)
    mask = (rng.random((T, 2)) < 0.5).astype(np.uint8)
    wide = np.zeros((T, max(new)), np.uint8)
    wide[:, :2] = mask
    q = p.rows(rng, 2)
    got = torch.full_like(q, 9.0)
    p.c.attention(0, q, got, 0.125, dev(mask, torch.uint8), stream=0)
    want, parts = p.m.attention(q.double().cpu().numpy(), 0.125, wide)
    assert (np.abs(got.double().cpu().numpy() - want) <= attention_bound("float32", want, parts, 64)).all()
    del g


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,new", [("float32", [130, 1]), ("bfloat16", [1, 150])])
def test_attention_behind_a_replayed_plan(gpu, dtype, new):
    """A prompt planned by a replay, after single tokens planned by a call: every row
    is written, by an eager call and by a graph that holds the attention alone; a
    graph of plan and attention for single tokens goes on beside them."""
    rng = np.random.default_rng(16)
    p = Pair(gpu, heads=4, kv_heads=2, hd=64, dtype=dtype)
    ctx = [70, 9]
    g = replayed_plan(p, ctx, new, 200, [1, 1], rng)
    q = p.rows(rng, 4)
    p.check_attention(q)
    out = torch.full_like(q, 9.0)
    s = torch.cuda.Stream()
    alone, both = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    pos, one = dev([a + b for a, b in zip(ctx, new)]), dev([1, 1])
    q1, k1 = q[:2].clone(), p.rows(rng, 2, 2)
    out1 = torch.full_like(q1, 9.0)
    torch.cuda.synchronize()
    with torch.cuda.graph(alone, stream=s):
        p.c.attention(0, q, out, stream=s.cuda_stream)
    with torch.cuda.graph(both, stream=s):
        p.c.plan(pos, one, 1, stream=s.cuda_stream)
        p.c.append(0, k1, k1, stream=s.cuda_stream)
        p.c.attention(0, q1, out1, stream=s.cuda_stream)
    torch.cuda.synchronize()
    alone.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, p.check_attention(q))
    both.replay()
    torch.cuda.synchronize()
    p.m.plan(pos.tolist(), [1, 1], 1)
    p.m.append(k1.double().cpu().numpy(), k1.double().cpu().numpy())
    want, parts = p.m.attention(q1.double().cpu().numpy(), 0.125)
    assert (np.abs(out1.double().cpu().numpy() - want) <= attention_bound(dtype, want, parts, 64)).all()
    del g


# ------------------------------------------------------------ V scales far apart
def check_small_values(p, q, small, mask=None):
    """Rows whose weight lies on keys with small V (at most `small`), beside keys of
    far larger V without weight. The scale of a block (in the kernel for many rows, of
    a page) is at least 2^-8 of the accumulators', so a probability's halves lose 2^-24
    of its own block's V instead of the 2^-31 of the largest V that attention_bound counts."""
    got = torch.full_like(q, 9.0)
    p.c.attention(0, q, got, 1.0, None if mask is None else dev(mask, torch.uint8), stream=0)
    want, (mag, smag, keys, vmax) = p.m.attention(q.double().cpu().numpy(), 1.0, mask)
    assert np.abs(want).max() <= small
    err = np.abs(got.double().cpu().numpy() - want)
    tol = attention_bound(p.dtype, want, (mag, smag, keys, np.full_like(vmax, 2.0 ** 7 * small)), p.hd)
    assert not np.isnan(err).any() and (err <= tol).all(), f"{(err / tol).max():.3g} x the bound"


@pytest.mark.gpu
@pytest.mark.parametrize("type", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("far,new,unit", [(-12, 6, BLOCK), (-20, 6, BLOCK), (-40, 6, BLOCK), (-12, 200, BLOCK),
                                          (-20, 200, PAGE), (-40, 200, PAGE)])
def test_values_of_scales_far_apart(gpu, far, new, unit, dtype, type):
    """Blocks (or pages) of keys with V near 1, which no row weighs (scores 60 lower:
    2^-86), among others with V near 2^far, in changing order; few rows and many."""
    rng = np.random.default_rng(-far)
    p = Pair(gpu, heads=2, kv_heads=1, hd=64, dtype=dtype, type=type, max_rows=1200, max_ctx=1200, pages=100)
    n = 1000
    large = rng.random((n + new) // unit + 1) < 0.4
    large[:3] = True, False, True
    large[-3:] = False, True, False
    large = np.repeat(large, unit)[:n + new]
    k = rng.standard_normal((n + new, 1, 64)) * 0.3
    k[:, :, 0] = np.where(large, -30.0, 30.0)[:, None]
    v = rng.uniform(-1, 1, (n + new, 1, 64)) * np.where(large, 1.0, 2.0 ** far)[:, None, None]
    k, v = (dev(x, torch.float32).to(getattr(torch, dtype)) for x in (k, v))
    q = p.rows(rng, 2, new)
    q[:, :, 0] = 1.0
    p.plan([0], [n])
    p.append(k[:n], v[:n])
    p.plan([n], [new])
    p.append(k[n:], v[n:])
    check_small_values(p, q, 2.0 ** far)


@pytest.mark.gpu
@pytest.mark.parametrize("far", [-20, -40])
@pytest.mark.parametrize("new,hidden", [(90, 2 * BLOCK), (200, PAGE)])
def test_unseen_values_of_larger_scales(gpu, far, new, hidden):
    """Large V in the first new rows, which the mask hides from every row."""
    rng = np.random.default_rng(17)
    p = Pair(gpu, heads=1, kv_heads=1, hd=64)
    p.plan([0], [new])
    k, v = rng.standard_normal((2, new, 1, 64))
    v = np.clip(v, -1, 1) * np.where(np.arange(new) < hidden, 1.0, 2.0 ** far)[:, None, None]
    p.append(dev(k, torch.float32), dev(v, torch.float32))
    mask = (rng.random((new, new)) < 0.5).astype(np.uint8)
    mask[:, :hidden] = 0
    mask[:, -1] = 1
    check_small_values(p, p.rows(rng, 1) * 0.3, 2.0 ** far, mask)


# -------------------------------------------- CTAs that take one tile after another
def ragged(kind, rng):
    """heads, kv_heads, hd, cached lengths, new rows: more (tile, kv head) pairs than
    CTAs, shared as whole tiles or, beside a few long sequences, as equal parts."""
    if kind == "rows-whole":
        return 32, 32, 32, rng.integers(0, 200, 48), rng.integers(1, 4, 48)
    if kind == "rows-parts":
        return 32, 16, 64, np.r_[rng.integers(0, 100, 60), 7000, 3000], rng.integers(1, 9, 62)
    if kind == "chunks-whole":
        return 16, 8, 64, rng.integers(0, 300, 24), rng.integers(97, 200, 24)
    if kind == "chunks-parts":
        return 16, 8, 64, np.r_[6000, rng.integers(0, 100, 20)], rng.integers(97, 150, 21)
    return 16, 8, 128, np.r_[rng.integers(0, 700, 20), 5000], np.r_[rng.integers(97, 150, 9), rng.integers(1, 40, 12)]


def check_in_bulk(p, q, mask=None):
    """check_attention with the model's formulas as 64-bit products on the GPU."""
    got = torch.full_like(q, 9.0)
    p.c.attention(0, q, got, None, None if mask is None else dev(mask, torch.uint8), stream=0)
    scale, r = float(np.float32(p.hd ** -0.5)), 0
    mk = None if mask is None else dev(mask, torch.bool)
    for b, m in enumerate(p.m.new):
        if not m:
            continue
        n, g = p.m.ctx[b] + m, p.H // p.Hk
        K, V = (dev(p.m.values(x, b), torch.float64) for x in "kv")
        x = q[r:r + m].double().view(m, p.Hk, g, p.hd)
        see = torch.arange(n, device="cuda")[None] <= p.m.ctx[b] + torch.arange(m, device="cuda")[:, None]
        if mk is not None:
            see[:, p.m.ctx[b]:] = mk[r:r + m, :m]
        see, any_ = see[:, None, None], see.any(1)[:, None, None]
        S = torch.einsum("mhgd,nhd->mhgn", x, K) * scale
        w = torch.where(any_[..., None], torch.where(see, S, -np.inf), 0.0).softmax(-1) * see
        want = torch.einsum("mhgn,nhd->mhgd", w, V)
        mag = torch.einsum("mhgn,nhd->mhgd", w, V.abs())
        smag = (torch.einsum("mhgd,nhd->mhgn", x.abs(), K.abs()) * see).amax(-1) * scale
        vmax = (V.abs().amax(-1).T[:, None] * see).amax(-1)
        keys = see.sum(-1).clamp(min=1)
        full = lambda a: a.expand(m, p.Hk, g).reshape(m, p.H).cpu().numpy()
        want, mag = (a.reshape(m, p.H, p.hd).cpu().numpy() for a in (want, mag))
        err = np.abs(got[r:r + m].double().cpu().numpy() - want)
        tol = attention_bound(p.dtype, want, (mag, full(smag), full(keys), full(vmax)), p.hd)
        assert not np.isnan(err).any() and (err <= tol).all(), f"{(err / np.maximum(tol, 1e-300)).max():.3g} x the bound"
        r += m
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,type", [("float32", "int8"), ("bfloat16", "e4m3"), ("float16", "int8")])
@pytest.mark.parametrize("kind", ["rows-whole", "rows-parts", "chunks-whole", "chunks-parts", "both"])
def test_more_tiles_than_ctas(gpu, kind, dtype, type):
    """Barriers, rings and workspaces carried from tile to tile within a CTA, with and
    without a mask; the same call again gives the same bits."""
    rng = np.random.default_rng(18)
    H, Hk, hd, ctx, new = ragged(kind, rng)
    pages = int((-(-(ctx + new) // PAGE)).sum())
    p = Pair(gpu, heads=H, kv_heads=Hk, hd=hd, dtype=dtype, type=type, pages=pages, max_seqs=len(ctx),
             max_rows=int(max(ctx.sum(), new.sum())), max_ctx=int((ctx + new).max()))
    p.plan([0] * len(ctx), ctx.tolist(), check=False)
    p.append(p.rows(rng, Hk, scale=2.0), p.rows(rng, Hk))
    p.plan(ctx.tolist(), new.tolist(), check=False)
    p.append(p.rows(rng, Hk, scale=2.0), p.rows(rng, Hk))
    q = p.rows(rng, H)
    first = check_in_bulk(p, q)
    for _ in range(5):
        out = torch.full_like(q, 9.0)
        p.c.attention(0, q, out, hd ** -0.5, stream=0)
        assert torch.equal(out, first)
    mask = (rng.random((int(new.sum()), int(new.max()))) < 0.5).astype(np.uint8)
    check_in_bulk(p, q, mask)
    p.c.attention(0, q, out, stream=0)
    assert torch.equal(out, first)
    assert gpu.fl_cuda_sync() == 0


@pytest.mark.gpu
def test_plans_refused_in_the_life_of_a_batch(gpu):
    """Steps of a running batch that lack pages, that have too many rows, and that go
    through, all of them among the steps."""
    rng = np.random.default_rng(1)
    p = Pair(gpu, pages=20, max_seqs=9, max_rows=300, max_ctx=500)
    pos, seen = np.zeros(9, int), []
    for step in range(60):
        new = np.minimum(rng.integers(0, 40, 9), 512 - pos)
        new[rng.random(9) < 0.1] = -1
        if step % 6 == 3:
            new[rng.integers(9)] = 260 if step % 4 == 1 else 150
        p.plan(pos.tolist(), new.tolist(), max_new=260)
        seen.append(p.m.status)
        if p.m.status == 0:
            pos = np.where(new < 0, 0, pos + np.maximum(new, 0))
        elif p.m.status > 0:                     # a scheduler makes room
            pos[:3] = 0
            p.plan(pos.tolist(), [-1] * 3 + [0] * 6, max_new=260)
            assert p.m.status == 0
    assert 0 in seen and -1 in seen and max(seen) > 0


# --------------------------------------------------------- sums over many keys
@pytest.mark.gpu
@pytest.mark.parametrize("type", ["int8", "e4m3"])
@pytest.mark.parametrize("seqs,kv_heads,hd,ctx,new", [(12, 40, 32, 30000, 1), (1, 40, 32, 30000, 1024), (1, 20, 128, 20000, 2048)])
def test_sums_over_many_keys_do_not_drift(gpu, seqs, kv_heads, hd, ctx, new, type):
    """f32 rows over tens of thousands of keys that one CTA takes in a row, V positive:
    sums that drop the bits below 2^-24 at each of n products fall short by about
    n 2^-25; rounded ones do not fall short on average. 2^-20 is 32 steps of 2^-25 left
    to the products of a few blocks, twice over. One value is off by at most that,
    2^-22 for its probabilities' halves, 2^-24 for each 16 keys, and the scores' errors,
    2^-20 of scores below 8."""
    n = ctx + new
    c = flb200.KV8Cache(gpu, layers=1, heads=kv_heads, kv_heads=kv_heads, head_dim=hd, pages=seqs * -(-n // PAGE),
                        max_seqs=seqs, max_rows=max(ctx, seqs * new), max_ctx=n, type=type, dtype="float32")
    g = torch.Generator(device="cuda").manual_seed(19)
    v = torch.rand((n, kv_heads, hd), generator=g, device="cuda") * 0.5 + 0.5
    k = torch.randn((n, kv_heads, hd), generator=g, device="cuda")
    for b in range(seqs):
        c.plan(dev([0] * seqs), dev([ctx if i == b else 0 for i in range(seqs)]), ctx, stream=0)
        c.append(0, k[:ctx], v[:ctx], stream=0)
    c.plan(dev([ctx] * seqs), dev([new] * seqs), new, stream=0)
    c.append(0, k[ctx:].repeat(seqs, 1, 1), v[ctx:].repeat(seqs, 1, 1), stream=0)
    q = torch.randn((new, kv_heads, hd), generator=g, device="cuda").repeat(seqs, 1, 1)
    out = torch.full_like(q, 9.0)
    c.attention(0, q, out, stream=0)
    gk, gv = (torch.empty((seqs * n, kv_heads, hd), device="cuda") for _ in range(2))
    c.gather(0, gk, gv, stream=0)
    hide = torch.arange(n, device="cuda") > ctx + torch.arange(new, device="cuda")[:, None]
    scale, rel = float(np.float32(hd ** -0.5)), []
    for h in range(0, kv_heads, 3):
        S = q[:new, h].double() @ gk[:n, h].double().T * scale
        assert S.abs().max() < 8
        want = S.masked_fill_(hide, -np.inf).softmax(1) @ gv[:n, h].double()
        rel.append((out[:, h].view(seqs, new, hd).double() - want) / want)
    rel = torch.stack(rel)
    assert abs(float(rel.mean())) <= 2.0 ** -20
    assert float(rel.abs().max()) <= 2.0 ** -20 + 2.0 ** -22 + n / 16 * 2.0 ** -24 + 2.0 ** -17
