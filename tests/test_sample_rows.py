"""fl_cuda_sample against the rule computed on the host: the oracle's integer
weights, then the filters and the draw in Python integers. Tokens are whole
numbers, so they have to be equal.

- CPU: refused arguments;
- GPU: types, vocabulary sizes on both sides of every CTA and cluster size,
  misaligned and strided rows, ties at the top-k boundary, rows with nothing,
  one or only equal logits, infinities and NaN, every parameter at its ends;
  a caller's stream and a captured graph."""
import numpy as np
import pytest

import flb200

ONE = 1 << 24


def test_refusals(lib):
    f = lib.fl_cuda_sample
    ok = dict(logits=64, dtype=0, ld=8, rows=1, V=8, t=None, k=None, p=None, m=None, u=64, tok=64, s=None)

    def rc(**kw):
        return f(*dict(ok, **kw).values())
    assert rc(rows=0, logits=None, u=None, tok=None) == 0          # nothing to do
    for kw in (dict(rows=-1), dict(V=0), dict(dtype=3), dict(dtype=-1), dict(logits=None), dict(u=None),
               dict(tok=None), dict(rows=2, ld=7), dict(logits=66), dict(dtype=1, logits=65)):
        assert rc(**kw) == -1, kw
        assert lib.err().startswith("sample: ")
    assert rc(V=262001, ld=262001) == -4


def test_misaligned_arrays_are_refused(lib):
    f = lib.fl_cuda_sample
    ok = dict(logits=64, dtype=0, ld=8, rows=1, V=8, t=64, k=64, p=64, m=64, u=64, tok=64, s=None)
    for name, arg in (("temperature", "t"), ("top_k", "k"), ("top_p", "p"), ("min_p", "m"), ("u", "u"), ("tokens", "tok")):
        for at in (65, 66):
            assert f(*dict(ok, **{arg: at}).values()) == -1
            assert lib.err() == f"sample: {name} is not aligned to its type"


def expect(orc, l, T, k, p, m, u):
    """The rule for one row of float32 logits."""
    l = np.where(np.isnan(l), -np.inf, np.minimum(l, np.finfo(np.float32).max)).astype(np.float32) + np.float32(0)
    if l.max() == -np.inf:
        return -1
    if not T > 0:
        return int(np.argmax(l))
    E, _ = orc.sample_weights(np.ascontiguousarray(l), float(T), 1.0)
    E = np.asarray(E).astype(np.int64)      # sums stay below 2^18 * 2^24
    if 1 <= k:
        E[np.argsort(-l, kind="stable")[k:]] = 0
    lo = 1
    if p < 1:
        P = max(1, int(np.float32(max(p, 0)) * np.float32(ONE)))
        s = np.sort(E)[::-1]
        c = np.cumsum(s)
        lo = max(1, int(s[np.searchsorted(c, -(-P * int(c[-1]) // ONE))]))
    lo = max(lo, int(np.float32(min(max(m, 0), 1)) * np.float32(ONE)))
    c = np.cumsum(np.where(E >= lo, E, 0))
    tgt = (min(int(np.float32(u) * np.float32(ONE)), ONE - 1) * int(c[-1])) >> 24
    return int(np.searchsorted(c, tgt, side="right"))


def run(gpu, logits, u, T=None, k=None, p=None, m=None, stream=None):
    import torch
    dev = lambda a, t: None if a is None else torch.tensor(np.asarray(a), dtype=t, device="cuda")
    out = torch.full((logits.shape[0],), -7, dtype=torch.int32, device="cuda")
    flb200.sample(gpu, logits, dev(u, torch.float32), out, dev(T, torch.float32), dev(k, torch.int32),
                  dev(p, torch.float32), dev(m, torch.float32), stream=0 if stream is None else stream)
    torch.cuda.synchronize()
    return out.cpu().numpy()


def check(gpu, orc, logits, u, T, k, p, m):
    got = run(gpu, logits, u, T, k, p, m)
    h = logits.float().cpu().numpy()
    R = len(h)
    full = lambda a, d: np.full(R, d) if a is None else np.asarray(a)
    # parameters as the float32 the device reads
    f32 = lambda a, d: full(a, d).astype(np.float32)
    for r in range(R):
        want = expect(orc, h[r], f32(T, 1.0)[r], int(full(k, 0)[r]), f32(p, 1.0)[r], f32(m, 0.0)[r], f32(u, 0)[r])
        assert got[r] == want, (r, got[r], want)


def make(rng, R, V, dtype, scale=3.0):
    import torch
    l = rng.standard_normal((R, V)) * scale
    return torch.tensor(l, device="cuda").to(getattr(torch, dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("V", [1, 2, 31, 1000, 8184, 8185, 32064])
def test_parameters(gpu, orc, dtype, V):
    rng = np.random.default_rng(V)
    R = 12
    l = make(rng, R, V, dtype)
    T = [0.7, 1.0, 1.3, 0.0, -1.0, np.nan, 0.05, 30.0, np.float32(1.9999999), 1.0, 0.9, 1e-25]
    k = [0, 5, V, 1, 7, 3, 50, V + 9, 40, 0, max(1, V // 2), 2]
    p = [0.9, 1.0, 0.5, 0.3, 0.2, 0.9, 0.999, 0.7, 0.0, 1e-9, 0.95, 0.5]
    m = [0.0, 0.05, 0.0, 0.5, 0.1, 0.0, 0.2, 0.9, 0.0, 0.001, 1.0, 0.0]
    u = rng.random(R).astype(np.float32)
    u[:2] = 0.0, np.float32(1 - 2 ** -24)
    check(gpu, orc, l, u, T, k, p, m)
    check(gpu, orc, l, u, None, k, None, None)
    check(gpu, orc, l, u, T, None, p, None)
    check(gpu, orc, l, u, None, None, None, m)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("V", [9000, 32064])
def test_many_rows(gpu, orc, dtype, V):
    """More rows than the GPU holds at four CTAs a row: one CTA each."""
    rng = np.random.default_rng(V)
    R = 160
    l = make(rng, R, V, dtype)
    check(gpu, orc, l, rng.random(R), rng.uniform(0.3, 1.5, R), rng.integers(0, 60, R), rng.uniform(0.2, 1.1, R),
          rng.uniform(0, 0.05, R))


def test_order_of_the_weights(tmp_path):
    """What the kernel's top-k relies on: weights are ordered as their logits but
    for differences of one between the two named constants (every float gone
    through in C)."""
    import os
    import shutil
    import subprocess
    if shutil.which("gcc") is None:
        pytest.skip("needs gcc")
    here = os.path.dirname(os.path.abspath(__file__))
    exe = tmp_path / "sample_weight_check"
    subprocess.run(["gcc", "-O3", "-march=native", "-ffp-contract=off", "-o", str(exe),
                    os.path.join(here, "sample_weight_check.c"), "-lm"], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=600, check=True)
    assert r.stdout == f"below 1 floats 2878 weights 13066122 to 16518617 largest {ONE}\n"
    src = open(os.path.join(os.path.dirname(flb200.LIB_PATH), "csrc", "sample_rows.cu")).read()
    assert "kUnorderedMin = 13066122u, kUnorderedMax = 16518617u" in src


@pytest.mark.gpu
@pytest.mark.parametrize("V", [3, 5000, 30000, 100000])
def test_top_k_is_by_logits(gpu, orc, V):
    """A pair of neighbouring logits of which the larger has the smaller weight,
    at the cut of top-k: alone (the other logits far below), and in a row so hot
    that the cut lies in a crowd of such weights."""
    import torch
    a, b = np.float32(-0.224945396), np.float32(-0.224945411)
    E, _ = orc.sample_weights(np.array([0, a, b], np.float32), 1.0, 1.0)
    assert a > b and E[1] < E[2]
    rng = np.random.default_rng(V)
    l = np.full((6, V), -9.0, np.float32)
    for r in range(6):
        l[r, rng.permutation(V)[:3]] = np.roll([0, a, b], r)
    d = torch.tensor(l, device="cuda")
    for u in (0.0, 0.3, 0.55, 0.9, 0.9999):
        for k in (1, 2, 3):
            for p in (None, [0.7] * 6, [0.99] * 6):
                check(gpu, orc, d, [u] * 6, None, [k] * 6, p, None)
    for dtype in ("float32", "bfloat16"):
        hot = make(rng, 6, V, dtype, 8.0)
        for T in (40.0, 150.0, 400.0):
            for k in (2, max(2, V // 3), V - 1):
                check(gpu, orc, hot, rng.random(6), [T] * 6, [k] * 6, None, None)
                check(gpu, orc, hot, rng.random(6), [T] * 6, [k] * 6, [0.8] * 6, [0.0, 0.9, 0.95, 0.0, 0.5, 1.0])
    # the cut within a crowd of one unordered pair's floats
    x = np.where(rng.random((6, V)) < 0.5, a, b).astype(np.float32)
    x[:, 0] = 0.0
    d = torch.tensor(x, device="cuda")
    for k in sorted({2, V // 2 + 1, V - 1}):
        check(gpu, orc, d, rng.random(6), None, [k] * 6, None, None)
    # weights next to each other of logits of both signs, far below the largest
    far = make(rng, 6, V, "float32", 3.0)
    far[:, 1] = 1e7
    for k in sorted({2, V // 2 + 1, V - 1}):
        check(gpu, orc, far, rng.random(6), [5e7] * 6, [k] * 6, None, None)


@pytest.mark.gpu
@pytest.mark.parametrize("R,V", [(160, 8000), (160, 20000), (8, 20000), (24, 60000), (12, 200000)])
def test_top_p_right_behind_a_small_top_k(gpu, orc, R, V):
    """At most 128 weights above the k-th: top-p then compares its weights all
    with all right after top-k did, in the same shared list. In every form
    (threads of a CTA, CTAs of a row), each call repeated."""
    import torch
    rng = np.random.default_rng(V)
    l = make(rng, R, V, "float32")
    k = rng.integers(2, 129, R)
    p = rng.uniform(0.3, 0.99, R)
    u = rng.random(R)
    check(gpu, orc, l, u, None, k, p, None)
    want = run(gpu, l, u, None, k, p)
    d = [torch.tensor(np.asarray(a), dtype=t, device="cuda") for a, t in ((u, torch.float32), (k, torch.int32), (p, torch.float32))]
    out = torch.empty((300, R), dtype=torch.int32, device="cuda")
    for o in out:
        flb200.sample(gpu, l, d[0], o, None, d[1], d[2], stream=0)
    assert (out.cpu().numpy() == want).all()


@pytest.mark.gpu
@pytest.mark.parametrize("V", [9000, 100000, 200000])
def test_clusters_that_start_one_after_another(gpu, orc, V):
    """More clusters than the GPU holds, on two streams at once: the CTAs of a
    row start whenever SMs fall free, next to other rows' ends."""
    import torch
    rng = np.random.default_rng(V)
    R = 70
    l = make(rng, R, V, "bfloat16")
    u = torch.tensor(rng.random(R), dtype=torch.float32, device="cuda")
    out = torch.empty((40, R), dtype=torch.int32, device="cuda")
    s = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for i, o in enumerate(out):
        flb200.sample(gpu, l, u, o, stream=s[i % 2].cuda_stream)
    torch.cuda.synchronize()
    h, hu = l.float().cpu().numpy(), u.cpu().numpy()
    want = [expect(orc, h[r], 1.0, 0, np.float32(1), np.float32(0), hu[r]) for r in range(R)]
    assert (out.cpu().numpy() == want).all()


@pytest.mark.gpu
def test_host_memory_is_refused(gpu):
    import torch
    l = torch.zeros((2, 100), device="cuda")
    t = torch.zeros(2, dtype=torch.int32, device="cuda")
    host = np.zeros((2, 100), np.float32)
    f = gpu.fl_cuda_sample
    assert f(flb200.ptr(host), 0, 100, 2, 100, None, None, None, None, l.data_ptr(), t.data_ptr(), None) == -1
    assert "not device memory" in gpu.err()
    assert f(l.data_ptr(), 0, 100, 2, 100, None, None, None, None, l.data_ptr(), flb200.ptr(host), None) == -1


@pytest.mark.gpu
def test_host_memory_of_any_array_is_refused(gpu):
    import torch
    l = torch.zeros((2, 100), device="cuda")
    t = torch.zeros(2, dtype=torch.int32, device="cuda")
    host = np.zeros(200, np.float32)
    names = ("temperature", "top_k", "top_p", "min_p", "u", "tokens")
    for i, name in enumerate(names):
        arr = [l.data_ptr()] * 5 + [t.data_ptr()]
        arr[i] = flb200.ptr(host)
        assert gpu.fl_cuda_sample(l.data_ptr(), 0, 100, 2, 100, *arr, None) == -1
        assert gpu.err() == f"sample: {name} is not device memory"
    assert gpu.fl_cuda_sync() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("V", [32760, 32761, 65520, 65521, 131072, 262000])
def test_clusters(gpu, orc, V):
    rng = np.random.default_rng(V)
    l = make(rng, 3, V, "bfloat16")
    check(gpu, orc, l, rng.random(3), [1.0, 0.8, 0.0], [0, 300, 0], [0.9, 0.95, 1.0], [0.0, 0.01, 0.0])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("V", [200, 9001, 40000])
def test_ties(gpu, orc, dtype, V):
    """Few different logits, so that top-k cuts through equal ones; weights
    that different logits share (far below the maximum); all equal."""
    import torch
    rng = np.random.default_rng(V)
    l = np.round(rng.standard_normal((4, V)) * 2) / 2
    l[1] = 1.25
    l[2] = -12 - rng.random(V) * 4      # weights of a few units
    l[2, V // 3] = 1.0
    l[3, ::3] = -np.inf
    l = torch.tensor(l, device="cuda").to(getattr(torch, dtype))
    for k in (1, 2, 63, V // 3, V - 1):
        check(gpu, orc, l, rng.random(4), None, [k] * 4, None, None)
        check(gpu, orc, l, rng.random(4), None, [k] * 4, [0.6] * 4, None)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("V", [500, 32064])
def test_logits_that_share_a_weight(gpu, orc, dtype, V):
    """Temperatures at which many different logits have the weight of the k-th:
    far below the maximum, or so hot that all are equal (keys of both signs)."""
    rng = np.random.default_rng(V)
    l = make(rng, 6, V, dtype, 2.0)
    l[:, 7] = 20.0
    for k in (1, 2, 40, V // 2, V - 1):
        check(gpu, orc, l, rng.random(6), [1.15, 0.9, 1e9, 1e15, 1e25, np.inf], [k] * 6, None, None)
        check(gpu, orc, l, rng.random(6), [1.15, 1e9, 1e9, 1e25, 1.0, 0.8], [k] * 6, [0.9999] * 6, None)


@pytest.mark.gpu
@pytest.mark.parametrize("V", [5, 3000, 33000])
def test_special_values(gpu, orc, V):
    import torch
    rng = np.random.default_rng(V)
    l = rng.standard_normal((8, V)).astype(np.float32)
    l[0] = -np.inf
    l[1] = np.nan
    l[2] = -np.inf
    l[2, V - 1] = -3.0
    l[3, 1] = np.inf
    l[4, :2] = np.inf
    l[5, 2] = np.nan
    l[6] = -3.4028235e38                 # the type's lowest value everywhere
    l[7] = -3.4028235e38
    l[7, 3] = -1e38
    d = torch.tensor(l, device="cuda")
    for T in (1.0, 0.0, np.inf, 1e-30):
        check(gpu, orc, d, rng.random(8), [T] * 8, [0, 0, 3, 0, 1, 4, 2, 0], [0.9] * 8, [0.1] * 8)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_strided_rows_and_untouched_neighbours(gpu, orc, dtype):
    """Rows of a wider buffer at every alignment: columns outside [off, off + V)
    hold larger logits, which must not be drawn."""
    import torch
    rng = np.random.default_rng(3)
    buf = make(rng, 5, 1031, dtype)
    V = 1000
    for off in range(0, 9):
        view = buf[:, off:off + V]
        wide = buf.clone()
        wide[:, :off] = 50.0
        wide[:, off + V:] = 50.0
        got = run(gpu, wide[:, off:off + V], [0.3] * 5, [0.9] * 5, [40] * 5, [0.9] * 5)
        assert np.array_equal(got, run(gpu, view.contiguous(), [0.3] * 5, [0.9] * 5, [40] * 5, [0.9] * 5))
        check(gpu, orc, view, [0.3] * 5, [0.9] * 5, [40] * 5, [0.9] * 5, None)


@pytest.mark.gpu
def test_top_p_alone_is_the_engine_rule(gpu, orc):
    rng = np.random.default_rng(9)
    l = make(rng, 6, 32064, "float32", 4.0)
    u = rng.random(6).astype(np.float32)
    got = run(gpu, l, u, [0.8] * 6, None, [0.95] * 6)
    for r in range(6):
        E, M = orc.sample_weights(l[r].cpu().numpy(), 0.8, 0.95)
        assert got[r] == orc.sample_pick(E, M, int(u[r] * np.float32(ONE)))


@pytest.mark.gpu
def test_stream_and_graph(gpu, orc):
    """A caller's stream, and a captured call replayed on new numbers."""
    import torch
    rng = np.random.default_rng(4)
    l = make(rng, 4, 32064, "float32")
    u = torch.tensor(rng.random(4), dtype=torch.float32, device="cuda")
    out = torch.zeros(4, dtype=torch.int32, device="cuda")
    tp = torch.full((4,), 0.9, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        flb200.sample(gpu, l, u, out, top_p=tp, stream=s.cuda_stream)
        with torch.cuda.graph(g, stream=s):
            flb200.sample(gpu, l, u, out, top_p=tp, stream=s.cuda_stream)
    for _ in range(3):
        u.copy_(torch.tensor(rng.random(4), dtype=torch.float32))
        l.copy_(make(rng, 4, 32064, "float32"))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        h, hu = l.cpu().numpy(), u.cpu().numpy()
        for r in range(4):
            assert int(out[r]) == expect(orc, h[r], 1.0, 0, np.float32(0.9), 0.0, hu[r])


def test_binding_refuses(lib):
    torch = pytest.importorskip("torch")
    l = torch.zeros((2, 8))
    with pytest.raises(flb200.FLError, match="device tensor"):
        flb200.sample(lib, l, l[:, 0], l[:, 0].int())
