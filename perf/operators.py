"""Cases, plain forms and 64-bit values of the ragged-batch serving operators.

One decoding step of a ragged batch over a paged KV cache held in 8 bits:

  plan       block tables, slot maps, row and key offsets from the request
             lengths (pages of 64 positions, taken from and returned to a
             stack of free pages)
  append     new K / V rows quantised into the cache, one power-of-two scale
             per 16 tokens and head, read back with gather as the values the
             codes stand for
  attention  query rows over that cache: one row a sequence, a few drafted
             rows, a masked tree, or a prompt chunk
  sample     one token per logits row: temperature, top-k, top-p and min-p,
             from given uniform numbers

`run` computes them with elementary torch operations, or, with `own` set,
calls this repository's library. Sizes: the 32 x 96 and 40 / 10 x 128 head
layouts, the 64-sequence batch with 7 verify rows, the 33-node draft tree and
the 32064-token vocabulary are this repository's benchmark configurations; the
others are generic.
"""
from __future__ import annotations

import math
import os
import sys
import zlib

import numpy as np
import torch

own = False

PAGE = 64     # positions per page
BLOCK = 16    # positions per scale
SUB = PAGE // BLOCK
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
DEV = "cuda"
ONE = 1 << 24


# ----------------------------------------------------------------- the cases
def listed():
    return [
        # a small decode batch: what every step of a lightly loaded server plans
        dict(name="plan-decode", op="plan", seqs=8, max_ctx=2048, new="one", turnover=False),
        # a large batch dropped and admitted anew, decodes and prompts mixed
        dict(name="plan-turnover", op="plan", seqs=1021, max_ctx=4096, new="mixed", turnover=True),
        # one new token for each of 64 sequences, appended inside part-filled scale blocks
        dict(name="append-decode", op="append", seqs=64, ctx_lo=1, ctx_hi=95, new_lo=1, new_hi=1, kv_heads=32,
             head_dim=96, dtype="f32", kv="int8"),
        # prompts of uneven lengths written in one call
        dict(name="append-prompts", op="append", seqs=6, ctx_lo=0, ctx_hi=0, new_lo=701, new_hi=4093, kv_heads=10,
             head_dim=128, dtype="bf16", kv="e4m3"),
        # one user, one token, a short context: latency alone
        dict(name="attn-one", op="attention", seqs=1, ctx_lo=129, ctx_hi=129, new_lo=1, new_hi=1, heads=32,
             kv_heads=32, head_dim=96, dtype="f32", kv="int8", mask="causal"),
        # the verify pass of a 64-sequence speculative batch (6 drafts and the last token)
        dict(name="attn-verify", op="attention", seqs=64, ctx_lo=1024, ctx_hi=1535, new_lo=7, new_hi=7, heads=32,
             kv_heads=32, head_dim=96, dtype="f32", kv="int8", mask="causal"),
        # single tokens over long contexts of very different lengths, grouped heads
        dict(name="attn-long", op="attention", seqs=24, ctx_lo=300, ctx_hi=32000, new_lo=1, new_hi=1, heads=40,
             kv_heads=10, head_dim=128, dtype="bf16", kv="int8", mask="causal"),
        # 33-node draft trees over the full context
        dict(name="attn-tree", op="attention", seqs=4, ctx_lo=3584, ctx_hi=3839, new_lo=33, new_hi=33, heads=40,
             kv_heads=10, head_dim=128, dtype="f16", kv="e4m3", mask="tree"),
        # prompt chunks behind cached prefixes (chunked prefill)
        dict(name="attn-chunk", op="attention", seqs=4, ctx_lo=0, ctx_hi=6000, new_lo=800, new_hi=2047, heads=32,
             kv_heads=8, head_dim=128, dtype="bf16", kv="int8", mask="causal"),
        # the token after a prompt, one user
        dict(name="sample-one", op="sample", rows=1, vocab=32064, dtype="f32", rule="nucleus"),
        # a 64-sequence batch with 7 verify rows, every request with its own parameters
        dict(name="sample-batch", op="sample", rows=448, vocab=32064, dtype="f32", rule="mixed"),
        # a wide vocabulary in 16 bits
        dict(name="sample-wide", op="sample", rows=61, vocab=128011, dtype="bf16", rule="topk"),
    ]


def _log(rng, lo, hi):
    """A whole number whose logarithm is uniform over [lo, hi]."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["plan", "append", "append", "attention", "attention", "attention", "sample", "sample"])
    if op == "plan":
        return dict(op=op, seqs=_log(rng, 1, 1021), max_ctx=_log(rng, 64, 4096), new=rng.choice(["one", "mixed"]),
                    turnover=rng.random() < 0.5)
    if op == "sample":
        vocab = _log(rng, 2, 128011)
        return dict(op=op, rows=_log(rng, 1, max(1, min(448, 14000000 // vocab))), vocab=vocab,
                    dtype=rng.choice(list(DTYPES)), rule=rng.choice(["nucleus", "mixed", "topk"]))
    hd = rng.choice([32, 64, 96, 128])
    kvh = _log(rng, 1, 40)
    if op == "append":
        new_hi = _log(rng, 1, 4093)
        seqs = _log(rng, 1, max(1, min(256, 15000000 // (new_hi * kvh * hd))))
        ctx_hi = _log(rng, 1, max(1, min(400, 15000000 // (seqs * kvh * hd))))
        return dict(op=op, seqs=seqs, ctx_lo=0, ctx_hi=ctx_hi, new_lo=rng.choice([0, 1, (new_hi + 1) // 2]),
                    new_hi=new_hi, kv_heads=kvh, head_dim=hd, dtype=rng.choice(list(DTYPES)),
                    kv=rng.choice(["int8", "e4m3"]))
    group = rng.choice([1, 2, 3, 4, 5, 7, 8])
    kvh = _log(rng, 1, max(1, 40 // group))
    form = rng.choice(["one", "few", "tree", "chunk"])
    new_hi = {"one": 1, "few": rng.randint(2, 16), "tree": rng.randint(5, 70), "chunk": _log(rng, 40, 2047)}[form]
    mask = "tree" if form == "tree" else "causal"
    ctx_hi = _log(rng, 1, 6000 if form in ("tree", "chunk") else 32000)
    # bounded by the listed cases' cache and arithmetic
    seqs = _log(rng, 1, max(1, min(128, 480000000 // ((ctx_hi + new_hi) * kvh * hd),
                                   int(8e10) // (new_hi * (ctx_hi + new_hi) * kvh * group * hd))))
    return dict(op=op, seqs=seqs, ctx_lo=rng.choice([0, ctx_hi // 2, ctx_hi]), ctx_hi=ctx_hi,
                new_lo=new_hi if form == "one" else rng.choice([0, 1, new_hi]) if form != "tree" else new_hi,
                new_hi=new_hi, heads=kvh * group, kv_heads=kvh, head_dim=hd, dtype=rng.choice(list(DTYPES)),
                kv=rng.choice(["int8", "e4m3"]), mask=mask)


# --------------------------------------------------------------- the inputs
def _lengths(case, seed):
    """Host lengths (cached, new) of every sequence: the case gives the pairs,
    the seed their order."""
    r = np.random.default_rng(zlib.crc32(repr(sorted((k, v) for k, v in case.items() if k != "name")).encode()))
    B = case["seqs"]
    if case["op"] == "plan":
        ctx = r.integers(0, case["max_ctx"], B)
        new = np.ones(B, np.int64)
        if case["new"] == "mixed":  # decodes, a few drafted rows, idle slots, some prompts
            kind = r.random(B)
            prompt = r.integers(1, max(2, case["max_ctx"] // 4), B)
            new = np.where(kind < 0.6, 1, np.where(kind < 0.8, r.integers(2, 9, B), np.where(kind < 0.9, 0, prompt)))
            new = np.minimum(new, case["max_ctx"] - ctx)
    else:
        ctx = r.integers(case["ctx_lo"], case["ctx_hi"] + 1, B)
        new = r.integers(case["new_lo"], case["new_hi"] + 1, B)
    new[0] = max(1, new[0])  # idle sequences among others, never alone
    order = np.random.default_rng([seed, 1]).permutation(B)
    return ctx[order].astype(np.int64), new[order].astype(np.int64)


def _pages(n):
    return (n + PAGE - 1) // PAGE


def _gen(seed, n):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed * 16 + n)
    return g


def _rows(seed, n, rows, heads, hd, dtype, spread):
    """Normal rows; with `spread`, a few channels are several times larger (as
    keys have) and rows differ in size."""
    g = _gen(seed, n)
    x = torch.randn((rows, heads, hd), generator=g, device=DEV, dtype=torch.float32)
    if spread:
        ch = torch.randn((1, heads, hd), generator=g, device=DEV)
        x *= torch.where(ch > 1.5, 5.0, 1.0)
        x *= 0.5 + torch.rand((rows, 1, 1), generator=g, device=DEV)
    return x.to(DTYPES[dtype])


def _tree_mask(B, M):
    """[B * M, M]: a chain with the other nodes hanging off it; node 0 is the
    root, odd nodes continue the chain, even ones are leaves."""
    par = [-1] + [max(0, i - 2 if i % 2 else i - 3) if i > 1 else 0 for i in range(1, M)]
    m = np.zeros((M, M), np.uint8)
    for i in range(M):
        j = i
        while j >= 0:
            m[i, j] = 1
            j = par[j]
    return torch.from_numpy(np.tile(m, (B, 1))).to(DEV)


def _free_stack(pages):
    """Stack of free pages: the top (end) is page 0."""
    return torch.arange(pages - 1, -1, -1, dtype=torch.int32, device=DEV)


def _tables(seqs, max_ctx, pages, max_rows):
    z = lambda *s: torch.zeros(s, dtype=torch.int32, device=DEV)
    return dict(block_table=z(seqs, max(1, _pages(max_ctx))), held=z(seqs), free_pages=_free_stack(pages),
                n_free=torch.full((1,), pages, dtype=torch.int32, device=DEV), row_start=z(seqs + 1),
                kv_start=z(seqs + 1), slot=z(max_rows), pos=z(max_rows), row_seq=z(max_rows), status=z(1))


def _lib():
    here = os.path.join(os.getcwd(), "fast-llm-inference_b200")
    if here not in sys.path:
        sys.path.insert(0, here)
    import flb200
    if not hasattr(_lib, "lib"):
        _lib.lib = flb200.Lib()
    return flb200, _lib.lib


def _stream():
    return torch.cuda.current_stream().cuda_stream


TABLES = ("block_table", "held", "free_pages", "n_free", "row_start", "kv_start", "slot", "pos", "row_seq", "status")


def prepare(case, seed):
    st = dict(case)
    op = case["op"]
    if op == "sample":
        return _prepare_sample(st, seed)
    ctx, new = _lengths(case, seed)
    B, T = case["seqs"], int(new.sum())
    dev = lambda a: torch.tensor(np.asarray(a), dtype=torch.int32, device=DEV)
    max_ctx = case["max_ctx"] if op == "plan" else int((ctx + new).max())
    max_ctx = max(1, max_ctx)
    pages = int(_pages(ctx + new).sum()) + 3
    st.update(ctx=ctx.tolist(), new=new.tolist(), dctx=dev(ctx), dnew=dev(new), max_new=max(1, int(new.max())), T=T)
    C = int(ctx.sum())
    # the prefix is planned as prompts; where no rows are appended, by its last positions alone
    pre = np.minimum(ctx, 1) if op == "plan" else ctx
    max_rows = max(T, int(pre.sum()))
    if op == "plan":
        st.update(kv_heads=1, head_dim=32, kv="int8", dtype="f32")
        st["drop"] = dev(np.full(B, -1))
    if own:
        flb200, lib = _lib()
        st["kv8"] = flb200.KV8Cache(lib, layers=1, heads=st.get("heads", st["kv_heads"]), kv_heads=st["kv_heads"],
                                    head_dim=st["head_dim"], pages=pages, max_seqs=B, max_rows=max_rows,
                                    max_ctx=max_ctx, type=st["kv"], dtype=str(DTYPES[st["dtype"]])[6:],
                                    device=torch.cuda.current_device())
        t = st["kv8"].tables()
        st["tables"] = {n: torch.as_tensor(t[n], device=DEV) for n in TABLES}
    else:
        st["tables"] = _tables(B, max_ctx, pages, max_rows)
    if own:
        st["kv8"].plan(dev(ctx - pre), dev(pre), max(1, int(pre.max())), stream=_stream())
    else:
        _plain_plan(st["tables"], dev(ctx - pre), dev(pre))
    if op == "plan":
        return st
    Hk, hd, dt = st["kv_heads"], st["head_dim"], st["dtype"]
    if not own:
        st["cache"] = _plain_cache(pages, Hk, hd, st["kv"])
    if C:
        k0, v0 = _rows(seed, 1, C, Hk, hd, dt, True), _rows(seed, 2, C, Hk, hd, dt, False)
        if own:
            st["kv8"].append(0, k0, v0, stream=_stream())
        else:
            _plain_append(st["cache"], st["tables"], k0, v0, C)
        del k0, v0
    st["k"], st["v"] = _rows(seed, 3, T, Hk, hd, dt, True), _rows(seed, 4, T, Hk, hd, dt, False)
    # the step's plan
    if own:
        st["kv8"].plan(st["dctx"], st["dnew"], st["max_new"], stream=_stream())
    else:
        _plain_plan(st["tables"], st["dctx"], st["dnew"])
    if op == "append":
        n = int((ctx + new)[new > 0].sum())
        if own:
            st["gk"] = torch.empty((n, Hk, hd), dtype=DTYPES[dt], device=DEV)
            st["gv"] = torch.empty_like(st["gk"])
        return st
    H = st["heads"]
    st["q"] = _rows(seed, 5, T, H, hd, dt, False)
    st["scale"] = 1.0 / math.sqrt(hd)
    st["mk"] = _tree_mask(B, st["new_hi"]) if st["mask"] == "tree" else None
    if own:
        st["kv8"].append(0, st["k"], st["v"], stream=_stream())
        st["out"] = torch.empty((T, H, hd), dtype=DTYPES[dt], device=DEV)
    else:
        _plain_append(st["cache"], st["tables"], st["k"], st["v"], T)
    return st


def _prepare_sample(st, seed):
    R, V = st["rows"], st["vocab"]
    g = _gen(seed, 1)
    r = np.random.default_rng([seed, 2])
    # logits as a language model's head gives them: a wide normal bulk, a few likely tokens
    l = torch.randn((R, V), generator=g, device=DEV) * 2.0
    n = min(V, 24)
    top = (torch.randint(0, V, (R, 1), generator=g, device=DEV) + torch.arange(n, device=DEV) * (V // n)) % V
    l.scatter_(1, top, 6.0 + 3.0 * torch.randn((R, n), generator=g, device=DEV))
    st["logits"] = l.to(DTYPES[st["dtype"]])
    f = lambda a: torch.tensor(np.asarray(a), dtype=torch.float32, device=DEV)
    st["u"] = torch.rand((R,), generator=g, device=DEV)
    st["temperature"] = f(r.uniform(0.5, 1.2, R))
    st["top_k"] = st["top_p"] = st["min_p"] = None
    if st["rule"] in ("nucleus", "mixed"):
        st["top_p"] = f(r.uniform(0.5, 0.99, R))
    if st["rule"] in ("topk", "mixed"):
        k = r.integers(1, 201, R)
        st["top_k"] = torch.tensor(k, dtype=torch.int32, device=DEV)
    if st["rule"] == "mixed":
        st["min_p"] = f(r.uniform(0.0, 0.1, R))
        for name, off in (("temperature", 0.0), ("top_k", 0), ("top_p", 1.0), ("min_p", 0.0)):
            st[name] = torch.where(torch.tensor(r.random(R) < 0.2, device=DEV), torch.full_like(st[name], off),
                                   st[name])
    if own:
        st["tokens"] = torch.empty((R,), dtype=torch.int32, device=DEV)
    return st


# --------------------------------------------------------------- the passes
def run(st):
    op = st["op"]
    if own:
        return _run_own(st)
    if op == "plan":
        if st["turnover"]:
            _plain_plan(st["tables"], st["dctx"], st["drop"])
        _plain_plan(st["tables"], st["dctx"], st["dnew"])
        return {n: st["tables"][n] for n in TABLES}
    if op == "append":
        # appended again, the same rows find their blocks' scales grown already: the same codes
        _plain_append(st["cache"], st["tables"], st["k"], st["v"], st["T"])
        return _plain_gather(st["cache"], st["tables"], st["ctx"], st["new"], DTYPES[st["dtype"]])
    if op == "attention":
        return _plain_attention(st)
    return _plain_sample(st)


def _run_own(st):
    s = _stream()
    op = st["op"]
    if op == "sample":
        flb200, lib = _lib()
        flb200.sample(lib, st["logits"], st["u"], st["tokens"], st["temperature"], st["top_k"], st["top_p"],
                      st["min_p"], stream=s)
        return st["tokens"]
    kv8 = st["kv8"]
    if op == "plan":
        if st["turnover"]:
            kv8.plan(st["dctx"], st["drop"], st["max_new"], stream=s)
        kv8.plan(st["dctx"], st["dnew"], st["max_new"], stream=s)
        return st["tables"]
    if op == "append":
        kv8.append(0, st["k"], st["v"], stream=s)
        kv8.gather(0, st["gk"], st["gv"], stream=s)
        return st["gk"], st["gv"]
    kv8.attention(0, st["q"], st["out"], st["scale"], st["mk"], stream=s)
    return st["out"]


# --------------------------------------------------- plan: pages and row maps
def _plan_pages(t, need, drop):
    """Returns the dropped sequences' pages to the stack (so that taking as
    many again gives each its old pages), then takes what `need` lacks, in
    (sequence, page) order. False where the pages do not suffice."""
    held, bt, n_free = t["held"].long(), t["block_table"], t["n_free"].long()
    B, mp = bt.shape
    j = torch.arange(mp, device=DEV)[None, :]
    rel = drop[:, None] & (j < held[:, None])
    keep = torch.where(drop, torch.zeros_like(held), held)
    take = (j >= keep[:, None]) & (j < need.long()[:, None])
    nrel, ntake = rel.sum(), take.sum()
    ok = (ntake <= n_free + nrel)[0] & (need.max() <= mp)
    # release: the first page of the first sequence ends on top
    free = torch.cat([t["free_pages"], t["free_pages"].new_zeros(1)])
    P = free.numel() - 1
    rr = rel.flatten().long().cumsum(0) - rel.flatten().long()
    dst = torch.where(rel.flatten() & ok, n_free + nrel - 1 - rr, torch.full_like(rr, P))
    free.scatter_(0, dst, bt.flatten())
    free = free[:P]
    top = n_free + nrel
    tr = take.flatten().long().cumsum(0) - take.flatten().long()
    src = (top - 1 - tr).clamp(0, P - 1)
    new_bt = torch.where(take.flatten() & ok, free[src], bt.flatten()).view(B, mp)
    t["free_pages"].copy_(torch.where(ok, free, t["free_pages"]))
    bt.copy_(new_bt)
    t["held"].copy_(torch.where(ok, torch.maximum(keep, need.long()), held))
    t["n_free"].copy_(torch.where(ok, top - ntake, n_free))
    missing = (ntake - top).clamp(min=0)
    t["status"].copy_(torch.where(ok, torch.zeros_like(missing), missing))
    return ok


def _plain_plan(t, ctx, new):
    drop = new < 0
    n = new.clamp(min=0).long()
    c = torch.where(drop, torch.zeros_like(ctx), ctx).long()
    tot = torch.where(n > 0, c + n, torch.zeros_like(c))     # idle sequences keep what they hold
    ok = _plan_pages(t, _pages(tot), drop)
    n = torch.where(ok, n, torch.zeros_like(n))
    tot = torch.where(ok & ~drop, c + n, torch.zeros_like(c))
    rs = torch.cat([n.new_zeros(1), n.cumsum(0)])
    t["row_start"].copy_(rs)
    t["kv_start"].copy_(torch.cat([n.new_zeros(1), torch.where(n > 0, tot, torch.zeros_like(tot)).cumsum(0)]))
    r = torch.arange(t["slot"].numel(), device=DEV)
    b = torch.searchsorted(rs[1:].contiguous(), r, right=True).clamp(max=n.numel() - 1)
    p = c[b] + r - rs[b]
    live = r < rs[-1]                                        # rows behind the last sequence stay as they are
    page = t["block_table"][b, (p // PAGE).clamp(0, t["block_table"].shape[1] - 1)].long()
    t["slot"].copy_(torch.where(live, page * PAGE + p % PAGE, t["slot"].long()))
    t["pos"].copy_(torch.where(live, p, t["pos"].long()))
    t["row_seq"].copy_(torch.where(live, b, t["row_seq"].long()))


# ------------------------------------------- append: power-of-two scales, codes
def _plain_cache(pages, Hk, hd, kv):
    c = dict(kv=kv)
    for n in "kv":
        c["c" + n] = torch.zeros((pages, Hk, SUB, BLOCK, hd), dtype=torch.int8 if kv == "int8" else torch.uint8,
                                 device=DEV)
        c["s" + n] = torch.zeros((pages, Hk, SUB), dtype=torch.float32, device=DEV)
    return c


def _pow2(e):
    """2^e as float32, -126 <= e <= 127."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _pow2_scale(amax, kv):
    """The smallest power of two s, at least 2^-100, with amax <= top * s, top
    the type's largest code: 127 = (127/128) 2^7, 448 = (7/8) 2^9."""
    m, x = torch.frexp(amax)
    lim, bits = (127.0 / 128.0, 7) if kv == "int8" else (0.875, 9)
    e = torch.where(m <= lim, x - bits, x - bits + 1).clamp(min=-100)
    return _pow2(torch.where(amax > 0, e, torch.full_like(e, -100)))


def _encode(y, kv):
    """Codes of values already divided by their scale."""
    y = torch.where(torch.isnan(y), torch.zeros_like(y), y)
    if kv == "int8":
        return y.clamp(-127, 127).round().to(torch.int8)
    return y.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)


def _decode(c, kv):
    return c.float() if kv == "int8" else c.view(torch.float8_e4m3fn).float()


def _plain_append(c, t, k, v, T):
    kv = c["kv"]
    slot = t["slot"][:T].long()
    page, sub, off = slot // PAGE, slot % PAGE // BLOCK, slot % BLOCK
    blk = page * SUB + sub
    r0 = t["row_start"][:-1].long().clamp(max=T - 1)     # only a sequence's first block can hold earlier tokens
    p0, b0 = page[r0], sub[r0]
    tok = torch.arange(BLOCK, device=DEV)[None, None, :, None]
    for n, x in (("k", k), ("v", v)):
        codes, scale = c["c" + n], c["s" + n]
        P, Hk, _, _, hd = codes.shape
        xf = x.float()
        a = torch.where(torch.isfinite(xf), xf.abs(), torch.zeros_like(xf)).amax(-1)           # [T, Hk]
        amax = a.new_zeros((P * SUB, Hk)).scatter_reduce_(0, blk[:, None].expand(T, Hk), a, "amax")
        first = off.new_full((P * SUB,), BLOCK).scatter_reduce_(0, blk, off, "amin")           # first new token
        amax = amax.view(P, SUB, Hk).transpose(1, 2)
        first = first.view(P, 1, SUB)
        s = _pow2_scale(amax, kv)
        s = torch.where(first < BLOCK, torch.where(first > 0, torch.maximum(s, scale), s), scale)
        # tokens that a touched block held before, in its new scale
        old = codes[p0, :, b0]
        ratio = (scale[p0, :, b0] / s[p0, :, b0])[..., None, None]
        codes[p0, :, b0] = torch.where(tok < first[p0, :, b0][..., None, None], _encode(_decode(old, kv) * ratio, kv), old)
        scale.copy_(s)
        codes[page, :, sub, off] = _encode(xf / s[page, :, sub][:, :, None], kv)


def _values(c, n, pages):
    """[tokens, Hk, hd] float32 values of whole pages."""
    x = _decode(c["c" + n][pages], c["kv"]) * c["s" + n][pages][..., None, None]
    m, Hk, _, _, hd = x.shape
    return x.permute(0, 2, 3, 1, 4).reshape(m * PAGE, Hk, hd)


def _plain_gather(c, t, ctx, new, dtype):
    return tuple(torch.cat([_values(c, n, t["block_table"][b, :_pages(cb + nb)].long())[:cb + nb].to(dtype)
                            for b, (cb, nb) in enumerate(zip(ctx, new)) if nb > 0]) for n in "kv")


# ------------------------------------------------------------------ attention
def _visible(cb, nb, b, st):
    """[nb, cb + nb] truth values: the cached positions, then the new rows at
    or before this one, or as the mask says."""
    if st["mk"] is None:
        i = torch.arange(nb, device=DEV)[:, None]
        return torch.arange(cb + nb, device=DEV)[None, :] <= cb + i
    m = st["mk"].view(st["seqs"], st["new_hi"], st["new_hi"])[b, :nb, :nb].bool()
    return torch.cat([torch.ones((nb, cb), dtype=torch.bool, device=DEV), m], 1)


def _plain_attention(st):
    q, c, t = st["q"], st["cache"], st["tables"]
    H, Hk, hd = st["heads"], st["kv_heads"], st["head_dim"]
    out = torch.empty_like(q)
    r = 0
    for b, (cb, nb) in enumerate(zip(st["ctx"], st["new"])):
        if nb == 0:
            continue
        n = cb + nb
        pages = t["block_table"][b, :_pages(n)].long()
        K = _values(c, "k", pages)[:n].permute(1, 2, 0)                # [Hk, hd, n]
        V = _values(c, "v", pages)[:n].permute(1, 0, 2)                # [Hk, n, hd]
        vis = _visible(cb, nb, b, st)
        g = H // Hk
        qb = q[r:r + nb].float().view(nb, Hk, g, hd).permute(1, 2, 0, 3).reshape(Hk, g * nb, hd)
        S = torch.matmul(qb, K).mul_(st["scale"]).view(Hk, g, nb, n)
        S.masked_fill_(~vis, -math.inf)
        m = S.amax(-1, keepdim=True)
        P = torch.exp(S - torch.where(m == -math.inf, torch.zeros_like(m), m))
        l = P.sum(-1, keepdim=True)
        o = torch.matmul(P.view(Hk, g * nb, n), V).view(Hk, g, nb, hd)
        o = torch.where(l > 0, o / l, torch.zeros_like(o))             # a row that sees nothing gives zeros
        out[r:r + nb] = o.permute(2, 0, 1, 3).reshape(nb, H, hd).to(out.dtype)
        r += nb
    return out


# ------------------------------------------------------------------- sampling
def _fma32(a, b, c):
    """a b + c rounded once to 32 bits (the product is exact in 64)."""
    return (a.double() * b.double() + c).float()


def _weights(x):
    """trunc(e^x 2^24) for x <= 0, 0 below -17, in the library's fixed
    sequence of correctly rounded operations (its sampling rule)."""
    f = lambda v: torch.tensor(v, dtype=torch.float32, device=x.device)
    xx = torch.where(x >= -17.0, x, torch.zeros_like(x))
    kf = torch.round(xx * f(1.442695))
    r = _fma32(-kf, f(0.693145751953125), xx.double())
    r = _fma32(-kf, f(1.4286068e-06), r.double())
    p = f(0.0001984127).expand_as(r)
    for co in (0.0013888889, 0.008333334, 0.041666668, 0.16666667, 0.5, 1.0, 1.0):
        p = _fma32(p, r, f(co).double())
    E = (p * _pow2(kf + 24)).long().clamp(max=ONE)      # an exact product
    return torch.where(x >= -17.0, E, torch.zeros_like(E))


def _fixed(p):
    """trunc(p 2^24) within [0, 2^24]."""
    return (p.clamp(0.0, 1.0) * float(ONE)).long()


def _split_mul(a, b, up):
    """floor (or, with up, ceil) of a b / 2^24 for a <= 2^24, b < 2^45."""
    lo = a * (b & (ONE - 1))
    return a * (b >> 24) + ((lo + (ONE - 1 if up else 0)) >> 24)


def _plain_sample(st):
    l = st["logits"].float()
    R, V = l.shape
    big = torch.finfo(torch.float32).max
    l = torch.where(torch.isnan(l), torch.full_like(l, -math.inf), l).clamp(max=big) + 0.0   # one zero
    mx = l.amax(1, keepdim=True)
    T = st["temperature"][:, None]
    hot = T > 0
    E = _weights(torch.where(mx > -math.inf, l - mx, torch.full_like(l, -math.inf)) /
                 torch.where(hot, T, torch.ones_like(T)))
    greedy = (l == mx).to(torch.int8).argmax(1)
    if st["top_k"] is not None:
        # the k largest logits, equal ones by index
        idx = torch.sort(l, dim=1, descending=True, stable=True)[1]
        rank = torch.empty_like(idx).scatter_(1, idx, torch.arange(V, device=DEV).expand(R, V))
        k = st["top_k"].long()[:, None]
        E = torch.where((k <= 0) | (rank < k), E, torch.zeros_like(E))
    keep = E > 0
    if st["top_p"] is not None:
        p = st["top_p"][:, None]
        P = _fixed(p).clamp(min=1)
        Es = torch.sort(E, dim=1, descending=True)[0]
        cum = Es.cumsum(1)
        need = _split_mul(P, cum[:, -1:], True)
        at = (cum < need).sum(1, keepdim=True).clamp(max=V - 1)
        keep = keep & ((p >= 1) | (E >= Es.gather(1, at)))
    if st["min_p"] is not None:
        keep = keep & (E >= _fixed(st["min_p"][:, None]))
    E = torch.where(keep, E, torch.zeros_like(E))
    cum = E.cumsum(1)
    U = (st["u"] * float(ONE)).long().clamp(0, ONE - 1)[:, None]
    tgt = _split_mul(U, cum[:, -1:], False)
    tok = (cum <= tgt).sum(1)
    tok = torch.where(hot[:, 0], tok, greedy)
    return torch.where(mx[:, 0] > -math.inf, tok, torch.full_like(tok, -1)).int()


# ------------------------------------------------------------------- the work
def work(case):
    op = case["op"]
    if op == "sample":
        eb = 4 if case["dtype"] == "f32" else 2
        n = case["rows"] * case["vocab"]
        return {"bytes": n * eb + case["rows"] * 24, "flops": 12 * n}
    ctx, new = _lengths(case, 0)
    T = int(new.sum())
    if op == "plan":
        pages = int(_pages(ctx + new).sum()) if case["turnover"] else int((new > 0).sum())
        return {"bytes": 4 * (3 * T + 7 * case["seqs"] + (4 if case["turnover"] else 1) * pages), "flops": 8 * T}
    eb = 4 if case["dtype"] == "f32" else 2
    w = case["kv_heads"] * case["head_dim"]
    n = int((ctx + new)[new > 0].sum())
    if op == "append":   # rows in, codes out, codes in, values out
        return {"bytes": 2 * w * (T * eb + T + n + n * eb) + 2 * case["kv_heads"] * 4 * (T + n) // BLOCK,
                "flops": 2 * w * (3 * T + n)}
    seen = int((new * ctx + (new * (new + 1) // 2 if case["mask"] == "causal" else new * new)).sum())
    return {"bytes": 2 * n * w + 2 * n * case["kv_heads"] * 4 // BLOCK + 2 * T * case["heads"] * case["head_dim"] * eb,
            "flops": 4 * seen * case["heads"] * case["head_dim"]}


# --------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    op = case["op"]
    keep = globals()["own"]
    globals()["own"] = False       # inputs only: nothing of the library
    try:
        return {"plan": _exact_plan, "append": _exact_append, "attention": _exact_attention,
                "sample": _exact_sample}[op](case, seed)
    finally:
        globals()["own"] = keep


def _exact_plan(case, seed):
    """The tables by their definition, request by request on the host."""
    ctx, new = _lengths(case, seed)
    B = case["seqs"]
    mp = max(1, _pages(case["max_ctx"]))
    pages = int(_pages(ctx + new).sum()) + 3
    pre = np.minimum(ctx, 1)
    max_rows = max(int(new.sum()), int(pre.sum()))
    slot, pos, seq = (np.zeros(max_rows, np.int64) for _ in range(3))
    stack = list(range(pages - 1, -1, -1))
    bt = np.zeros((B, mp), np.int64)
    held = np.zeros(B, np.int64)
    full = np.array(stack, np.int64)

    def grow(need):
        for b in range(B):
            while held[b] < need[b]:
                bt[b, held[b]] = stack.pop()
                held[b] += 1

    def rows(c, n):
        b = np.repeat(np.arange(B), n)
        p = c[b] + np.arange(len(b)) - np.repeat(np.cumsum(n) - n, n)
        slot[:len(b)], pos[:len(b)], seq[:len(b)] = bt[b, p // PAGE] * PAGE + p % PAGE, p, b
    grow(_pages(ctx))
    rows(ctx - pre, pre)
    if case["turnover"]:
        for b in range(B - 1, -1, -1):
            for j in range(held[b] - 1, -1, -1):
                stack.append(bt[b, j])
            held[b] = 0
        full[:len(stack)] = stack
    grow([_pages(c + n) if n > 0 else 0 for c, n in zip(ctx, new)])
    rows(ctx, new)
    rs = np.concatenate([[0], np.cumsum(new)])
    ks = np.concatenate([[0], np.cumsum(np.where(new > 0, ctx + new, 0))])
    res = dict(block_table=bt, held=held, free_pages=full, n_free=np.array([len(stack)]), row_start=rs, kv_start=ks,
               slot=slot, pos=pos, row_seq=seq, status=np.zeros(1, np.int64))
    return {n: torch.tensor(res[n], device=DEV).int() for n in TABLES}


def _round_e4m3(y):
    ex = torch.frexp(y.abs())[1].double() - 1.0
    q = torch.exp2(ex.clamp(min=-6.0)) / 8.0
    return torch.round(y / q) * q


def _coded(x, cb, kv):
    """[n, Hk, hd] float64 values that one sequence's rows stand for when its
    first cb rows are appended at once and the others after them: a block's
    scale covers its rows so far, and rows coded earlier are rounded again
    when it grows."""
    top = 127.0 if kv == "int8" else 448.0
    code = torch.round if kv == "int8" else _round_e4m3

    def scale(rows):  # of the largest value: ceil(log2(amax / top)) without a logarithm
        m, e = torch.frexp(rows.abs().amax((1, 3), keepdim=True) / top)
        return torch.where(m == 0.0, torch.full_like(e, -100), torch.where(m == 0.5, e - 1, e)).clamp(min=-100)
    n, Hk, hd = x.shape
    xb = torch.nn.functional.pad(x, (0, 0, 0, 0, 0, -n % BLOCK)).view(-1, BLOCK, Hk, hd)
    i = torch.arange(xb.shape[0] * BLOCK, device=x.device).view(-1, BLOCK, 1, 1)
    early, none = i < cb, torch.zeros_like(xb)
    e0 = scale(torch.where(early, xb, none))
    e1 = scale(torch.where(early, none, xb))
    e1 = torch.where(early.any(1, keepdim=True), torch.maximum(e0, e1), e1)
    e1 = torch.where((~early & (i < n)).any(1, keepdim=True), e1, e0)
    p2 = lambda e: ((e.long() + 1023) << 52).view(torch.float64)
    c0 = code(torch.where(early, xb, none) / p2(e0))
    c0 = torch.where(e1 > e0, code(c0 * p2(e0 - e1)), c0)
    val = torch.where(early, c0, code(xb / p2(e1))) * p2(e1)
    return val.view(-1, Hk, hd)[:n]


def _exact_rows(case, seed):
    """For every sequence with new rows: cached and new lengths and the
    float64 values of its K and V rows."""
    ctx, new = _lengths(case, seed)
    Hk, hd, dt = case["kv_heads"], case["head_dim"], case["dtype"]
    C, T = int(ctx.sum()), int(new.sum())
    raw = [(_rows(seed, n0, C, Hk, hd, dt, sp), _rows(seed, n1, T, Hk, hd, dt, sp))
           for n0, n1, sp in ((1, 3, True), (2, 4, False))]
    i = j = 0
    for cb, nb in zip(ctx.tolist(), new.tolist()):
        if nb > 0:
            yield cb, nb, [_coded(torch.cat([a[i:i + cb], b[j:j + nb]]).double(), cb, case["kv"]) for a, b in raw]
        i, j = i + cb, j + nb


def _exact_append(case, seed):
    vals = [kv for _, _, kv in _exact_rows(case, seed)]
    return tuple(torch.cat([kv[i] for kv in vals]) for i in range(2))


def _exact_attention(case, seed):
    H, Hk, hd = case["heads"], case["kv_heads"], case["head_dim"]
    T = int(_lengths(case, seed)[1].sum())
    q = _rows(seed, 5, T, H, hd, case["dtype"], False).double()
    tree = _tree_mask(1, case["new_hi"]).bool() if case["mask"] == "tree" else None
    out = torch.zeros((T, H, hd), dtype=torch.float64, device=DEV)
    r = 0
    for cb, nb, (k, v) in _exact_rows(case, seed):
        key = torch.arange(cb + nb, device=DEV)[None, :]
        for r0 in range(0, nb, 256):
            r1 = min(nb, r0 + 256)
            hide = key > cb + torch.arange(r0, r1, device=DEV)[:, None]
            if tree is not None:
                hide = torch.zeros_like(hide)
                hide[:, cb:] = ~tree[r0:r1, :nb]
            for h in range(H):
                s = q[r + r0:r + r1, h] @ k[:, h * Hk // H].T / math.sqrt(hd)
                s[hide] = -math.inf
                out[r + r0:r + r1, h] = torch.softmax(s, -1) @ v[:, h * Hk // H]
        r += nb
    return out


def _exact_sample(case, seed):
    """The rule row by row on the host, its exponentials in 64 bits."""
    if case["rows"] * case["vocab"] > 2e7:
        return None
    st = _prepare_sample(dict(case), seed)
    L = st["logits"].double().cpu().numpy()
    get = lambda n: None if st[n] is None else st[n].double().cpu().numpy()
    T, tk, tp, mp, u = get("temperature"), get("top_k"), get("top_p"), get("min_p"), get("u")
    out = np.zeros(case["rows"], np.int64)
    for r in range(case["rows"]):
        l = L[r]
        if not T[r] > 0:
            out[r] = int(l.argmax())
            continue
        x = (l - l.max()) / T[r]
        E = np.where(x >= -17.0, np.floor(np.exp(np.maximum(x, -18.0)) * ONE), 0.0).astype(np.int64)
        if tk is not None and tk[r] > 0:
            order = np.argsort(-l, kind="stable")
            E[order[int(tk[r]):]] = 0
        keep = E > 0
        if tp is not None and tp[r] < 1:
            P = max(1, int(np.floor(tp[r] * ONE)))
            s = np.sort(E)[::-1]
            c = np.cumsum(s)
            need = (P * int(c[-1]) + ONE - 1) // ONE
            keep &= E >= s[min(len(s) - 1, int(np.searchsorted(c, need)))]
        if mp is not None:
            keep &= E >= int(np.floor(mp[r] * ONE))
        E[~keep] = 0
        c = np.cumsum(E)
        out[r] = int(np.searchsorted(c, (int(u[r] * ONE) * int(c[-1])) >> 24, side="right"))
    return torch.tensor(out, device=DEV).int()
