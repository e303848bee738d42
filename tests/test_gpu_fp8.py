"""Products with E4M3 weights and block scales against 64-bit sums of the same bytes; tolerances: fp8_ref.product."""
import numpy as np
import pytest

import fp8_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx(pkg):
    c = pkg.Context(pkg.synth.Dims(), n_layer=1, max_tokens=16, device=0)
    yield c
    c.close()


def _dev(ctx, *arrays):
    return [None if a is None else ctx.to_device(np.ascontiguousarray(a)) for a in arrays]


def _free(*bufs):
    for b in bufs:
        if b is not None:
            b.free()


def _quantize(ctx, x):
    n, K = x.shape
    d_x, = _dev(ctx, x)
    d_q, d_s = ctx.alloc(n * K), ctx.alloc(n * ref.blocks(K) * 4)
    ctx.fp8_quantize(d_x, n, K, d_q, d_s)
    got = d_q.download(np.uint8, (n, K)), d_s.download(np.float32, (n, ref.blocks(K)))
    _free(d_x, d_q, d_s)
    return got


@pytest.mark.parametrize("n,K", [(1, 16), (1, 2048), (3, 144), (5, 112), (130, 512), (7, 4096)])
def test_quantize_bit_exact(ctx, n, K):
    rng = np.random.default_rng(n * 10000 + K)
    x = (rng.standard_normal((n, K)) * np.exp2(rng.integers(-20, 20, (n, 1)))).astype(np.float32)
    x[0, :8] = [0.0, -0.0, 448.0, -448.0, 1e-3, 2.0**-9, 2.0**-10, 3 * 2.0**-11]
    q, s = _quantize(ctx, x)
    want_q, want_s = ref.quantize(x)
    assert np.array_equal(s, want_s) and np.array_equal(q, want_q)


def test_quantize_extremes(ctx):
    """Zeros, the smallest and the largest floats, infinities and NaN: those alone become NaN codes, and no scale notices them."""
    x = np.zeros((8, 256), np.float32)
    x[1, :4] = [1e-45, -1e-45, 3e-40, 1e-38]
    x[2, 0], x[2, 200] = 3.4028235e38, -3.4e38
    x[3, :3] = [np.inf, 5.0, -np.inf]
    x[4, 130] = np.nan
    x[5, :] = np.nan
    x[6, :] = 449.0
    x[7, :] = np.nextafter(np.float32(448), np.float32(1e9))
    q, s = _quantize(ctx, x)
    want_q, want_s = ref.quantize(x)
    nan = (want_q & 127) == 127
    assert np.array_equal(s, want_s) and np.array_equal((q & 127) == 127, nan) and np.array_equal(q[~nan], want_q[~nan])


def _gemm(ctx, w, ws, q, s):
    M, (n, K) = w.shape[0], q.shape
    d = _dev(ctx, w, ws, q, s)
    guard = np.full(n * M + 64, -7.25, np.float32)
    d_y, = _dev(ctx, guard)
    ctx.fp8_gemm(*d, d_y, M, K, n)
    ctx.sync()
    y = d_y.download(np.float32, n * M + 64)
    _free(*d, d_y)
    assert np.all(y[n * M:] == -7.25)                 # nothing behind the last row
    return y[:n * M].reshape(n, M)


SIZES = [(1, 1, 16), (1, 4096, 2048), (1, 257, 4096), (2, 130, 272), (5, 16, 128), (8, 100, 144), (9, 512, 640), (16, 2048, 4096), (17, 384, 1040), (31, 129, 2048),
         (33, 640, 512), (64, 1000, 256), (77, 1000, 1040), (128, 256, 2048), (129, 257, 144), (200, 4096, 512), (256, 8, 2176), (300, 130, 4096), (511, 1111, 528),
         (1000, 512, 2048)]


@pytest.mark.parametrize("n,M,K", SIZES)
def test_gemm(ctx, n, M, K):
    rng = np.random.default_rng(n + 7 * M + 13 * K)
    w, ws = ref.weights(rng, M, K)
    q = rng.integers(0, 256, (n, K)).astype(np.uint8)          # every code but NaN
    q[(q & 127) == 127] = 1
    s = rng.uniform(0.5, 3, (n, ref.blocks(K))).astype(np.float32)
    y = _gemm(ctx, w, ws, q, s)
    want, bound = ref.product(w, ws, q, s)
    assert np.all(np.abs(y - want) <= bound), np.max(np.abs(y - want) / bound)
    assert np.array_equal(y, _gemm(ctx, w, ws, q, s))          # the order of the sums is fixed


@pytest.mark.parametrize("n", [1, 12, 40, 130, 300])
def test_gemm_nan_and_zero_scales(ctx, n):
    """A NaN code in a weight row or an activation row spoils that row alone; scales of zero, an infinity and negative ones are numbers like others."""
    rng = np.random.default_rng(n)
    M, K = 300, 400
    w, ws = ref.weights(rng, M, K)
    q, s = ref.quantize(rng.standard_normal((n, K)).astype(np.float32))
    w[77, 390] = 127
    w[299, 0] = 255
    q[n // 2, 130] = 127
    ws[0, 1], s[n - 1, 2], ws[1, 0] = 0, 0, -0.01
    y = _gemm(ctx, w, ws, q, s)
    want, bound = ref.product(w, ws, q, s)
    assert np.array_equal(np.isnan(y), np.isnan(want))
    there = ~np.isnan(want)
    assert np.all(np.abs(y - want)[there] <= bound[there])


@pytest.mark.parametrize("n", [3, 70, 260])
def test_gemm_large_block_beside_small_ones(ctx, n):
    """One column block 2^30 above the others, then cancelled by a second one: the sums keep what f32 sums keep."""
    rng = np.random.default_rng(5)
    M, K = 128, 512
    w, ws = ref.weights(rng, M, K)
    w[:, 128:256] = w[:, :128]
    q, s = ref.quantize(rng.standard_normal((n, K)).astype(np.float32))
    q[:, 128:256] = q[:, :128] ^ 128
    s[:, 1] = s[:, 0]
    ws[:, 0] = ws[:, 1] = 2.0**20
    y = _gemm(ctx, w, ws, q, s)
    want, bound = ref.product(w, ws, q, s)
    assert np.all(np.abs(y - want) <= bound)


def test_gemm_tensor_core_sums(ctx):
    """What is lost of small products beside a large one inside a block of 128: at most 2^-23 of the sum a product, in every path."""
    for n in (4, 40, 200):
        M, K = 128, 128
        w = np.full((M, K), ref.encode(1.0), np.uint8)
        ws = np.ones((1, 1), np.float32)
        q = np.full((n, K), 1, np.uint8)                       # 2^-9
        q[:, 0] = 126                                          # 448
        s = np.ones((n, 1), np.float32)
        y = _gemm(ctx, w, ws, q, s)
        want, bound = ref.product(w, ws, q, s)
        assert np.all(np.abs(y - want) <= bound), (n, y[0, 0], want[0, 0])


def test_gemm_edges_and_refusals(ctx, pkg):
    d = ctx.alloc(1 << 16)
    before = ctx.launch_count()
    ctx.fp8_gemm(d, d, d, d, d, 16, 128, 0)                    # no rows: nothing is launched
    ctx.fp8_gemm(d, d, d, d, d, 0, 128, 4)
    ctx.fp8_quantize(d, 0, 128, d, d)
    assert ctx.launch_count() == before
    for bad in (lambda: ctx.fp8_gemm(d, d, d, d, d, 16, 0, 1), lambda: ctx.fp8_gemm(d, d, d, d, d, 16, 100, 1), lambda: ctx.fp8_gemm(d.ptr + 8, d, d, d, d, 16, 128, 1),
                lambda: ctx.fp8_gemm(d, d, d.ptr + 4, d, d, 16, 128, 1), lambda: ctx.fp8_gemm(d, None, d, d, d, 16, 128, 1), lambda: ctx.fp8_quantize(d, 1, 24, d, d),
                lambda: ctx.fp8_quantize(d.ptr + 4, 1, 16, d, d), lambda: ctx.fp8_quantize(d, 1, 16, None, d)):
        with pytest.raises(pkg.QkmError) as ei:
            bad()
        assert ei.value.code == -1
    with pytest.raises(pkg.QkmError) as ei:
        ctx.fp8_gemm(d, d, d, d, d, 16, 128, 1 << 28)
    assert ei.value.code == -3
    assert ctx.launch_count() == before
    d.free()


def _selection(rng, T, E, k, skew=0.0):
    """Selection records with distinct experts a token, and their pairs by expert."""
    from qwen_kernel_b200 import SEL_DTYPE
    sel = np.zeros(T, SEL_DTYPE)
    for t in range(T):
        p = np.exp(-skew * np.arange(E))
        sel["ids"][t, :k] = rng.choice(E, k, replace=False, p=p / p.sum())
        sel["w"][t, :k] = rng.dirichlet(np.ones(k))
        sel["w_shared"][t] = rng.uniform()
    e = sel["ids"][:, :k].reshape(-1)
    order = np.argsort(e, kind="stable")
    pairs = ((order // k) << 4 | order % k).astype(np.uint32)
    offsets = np.concatenate([[0], np.cumsum(np.bincount(e, minlength=E))]).astype(np.uint32)
    return sel, offsets, pairs


def _silu(g):
    return g / (1 + np.exp(-g))


def _swiglu_bound(g, u, bg, bu):
    """First order, with |d silu/dg| <= 1.1 and |silu(g)| <= |g|; expf, the quotient and the product: 2^-20 of the result."""
    return 1.1 * bg * (np.abs(u) + bu) + np.abs(g) * bu + bg * bu + 2.0**-20 * np.abs(_silu(g) * u)


def _experts_case(pkg, T, E, k, D, F, skew=0.0, seed=0, first=0, count=0):
    rng = np.random.default_rng(seed)
    dims = pkg.synth.Dims(n_embd=D, n_ff=F, n_expert=E, n_used=k)
    sel, offsets, pairs = _selection(rng, T, E, k, skew)
    x = rng.standard_normal((T, D)).astype(np.float32)
    h = rng.standard_normal((T * (k + 1), F)).astype(np.float32)
    mats = [ref.weights(rng, *shape, mats=E) for shape in ((F, D), (F, D), (D, F))]
    return dims, sel, offsets, pairs, ref.quantize(x), ref.quantize(h), mats


EXPERTS = [(1, 8, 2, 256, 256, 0.0), (1, 60, 4, 512, 256, 0.0), (5, 16, 4, 256, 512, 0.0), (16, 32, 8, 512, 256, 0.3), (33, 4, 3, 256, 256, 0.0), (100, 8, 2, 768, 256, 1.5),
           (300, 6, 2, 256, 256, 0.0), (150, 2, 2, 1280, 256, 0.0), (64, 512, 10, 256, 256, 0.0), (20, 17, 16, 256, 256, 0.0)]


@pytest.mark.parametrize("T,E,k,D,F,skew", EXPERTS)
def test_experts_grouped(pkg, T, E, k, D, F, skew):
    """gate/up and down by expert: experts without pairs, with one, with more than a tile; slots that no list names keep what they held."""
    dims, sel, offsets, pairs, (q, s), (hq, hs), ((g, gs), (u, us), (d, ds)) = _experts_case(pkg, T, E, k, D, F, skew, seed=T + E)
    with pkg.Context(dims, n_layer=1, max_tokens=1, device=0) as c:
        dev = _dev(c, g, gs, u, us, q, s, offsets, pairs, np.full((T, k + 1, F), 9.5, np.float32))
        c.moe_gateup_grouped_fp8(*dev, T)
        c.sync()
        h = dev[-1].download(np.float32, (T, k + 1, F))
        _free(*dev)
        dev = _dev(c, d, ds, hq, hs, sel, offsets, pairs, np.full((T, k, D), 9.5, np.float32))
        c.moe_down_grouped_fp8(*dev, T)
        c.sync()
        contrib = dev[-1].download(np.float32, (T, k, D))
        _free(*dev)
    assert np.all(h[:, k] == 9.5)
    for t in range(T):
        for j in range(k):
            e = sel["ids"][t, j]
            (wg, bg), (wu, bu) = (ref.product(m[e], ms[e], q[t:t + 1], s[t:t + 1]) for m, ms in ((g, gs), (u, us)))
            assert np.all(np.abs(h[t, j] - _silu(wg) * wu) <= _swiglu_bound(wg, wu, bg, bu)), (t, j, e)
            r = t * (k + 1) + j
            wd, bd = ref.product(d[e], ds[e], hq[r:r + 1], hs[r:r + 1])
            w = np.float64(sel["w"][t, j])
            assert np.all(np.abs(contrib[t, j] - w * wd) <= w * bd + 2.0**-23 * np.abs(w * wd)), (t, j, e)


@pytest.mark.parametrize("T", [1, 6, 40, 150, 300])
def test_shared_expert(pkg, T):
    rng = np.random.default_rng(T)
    D, F, k = 512, 256, 4
    dims = pkg.synth.Dims(n_embd=D, n_ff=F, n_expert=8, n_used=k)
    sel, _, _ = _selection(rng, T, 8, k)
    (g, gs), (u, us), (d, ds) = ref.weights(rng, F, D), ref.weights(rng, F, D), ref.weights(rng, D, F)
    q, s = ref.quantize(rng.standard_normal((T, D)).astype(np.float32))
    hq, hs = ref.quantize(rng.standard_normal((T * (k + 1), F)).astype(np.float32))
    with pkg.Context(dims, n_layer=1, max_tokens=1, device=0) as c:
        dev = _dev(c, g, gs, u, us, q, s, np.full((T, k + 1, F), 9.5, np.float32))
        c.moe_shared_gateup_fp8(*dev, T)
        c.sync()
        h = dev[-1].download(np.float32, (T, k + 1, F))
        _free(*dev)
        dev = _dev(c, d, ds, hq, hs, sel, np.zeros((T, D), np.float32))
        c.moe_shared_down_fp8(*dev, T)
        c.sync()
        y2 = dev[-1].download(np.float32, (T, D))
        _free(*dev)
    assert np.all(h[:, :k] == 9.5)
    (wg, bg), (wu, bu) = ref.product(g, gs, q, s), ref.product(u, us, q, s)
    assert np.all(np.abs(h[:, k] - _silu(wg) * wu) <= _swiglu_bound(wg, wu, bg, bu))
    at = np.arange(T) * (k + 1) + k
    wd, bd = ref.product(d, ds, hq[at], hs[at])
    w = sel["w_shared"].astype(np.float64)[:, None]
    assert np.all(np.abs(y2 - w * wd) <= w * bd + 2.0**-23 * np.abs(w * wd))


@pytest.mark.parametrize("T", [7, 90])
def test_lists_with_strangers(pkg, T):
    """Pairs that name a token or a slot that there is none of, offsets that end past the list or run backwards: the rest is computed."""
    E, k, D, F = 4, 2, 256, 256
    dims, sel, offsets, pairs, (q, s), (hq, hs), ((g, gs), (u, us), (d, ds)) = _experts_case(pkg, T, E, k, D, F, seed=3)
    good = np.ones(pairs.size, bool)
    for i, v in ((0, T << 4), (3, 0xFFFFFFF0), (5, 0 << 4 | 2), (pairs.size - 1, 15)):
        pairs[i], good[i] = v, False
    offsets[2] = offsets[1]                                    # expert 1 has none; its pairs go to nobody ...
    last = offsets[4]
    offsets[3], offsets[4] = last, last + 1000                 # ... expert 2 has the rest, the last offset is past the list
    owner = np.full(pairs.size, -1)
    for e in range(E):
        owner[offsets[e]:min(offsets[e + 1], pairs.size)] = e
    with pkg.Context(dims, n_layer=1, max_tokens=1, device=0) as c:
        dev = _dev(c, d, ds, hq, hs, sel, offsets, pairs, np.full((T, k, D), 9.5, np.float32))
        c.moe_down_grouped_fp8(*dev, T)
        c.sync()
        contrib = dev[-1].download(np.float32, (T, k, D))
        _free(*dev)
    want = np.full((T, k, D), 9.5)
    for p in np.flatnonzero(good & (owner >= 0)):
        t, j = pairs[p] >> 4, pairs[p] & 15
        r = t * (k + 1) + j
        want[t, j] = ref.product(d[owner[p]], ds[owner[p]], hq[r:r + 1], hs[r:r + 1])[0][0] * sel["w"][t, j]
    assert np.array_equal(contrib == 9.5, want == 9.5)
    assert np.allclose(contrib, want, rtol=1e-4, atol=1e-4 * np.abs(want).max())


def test_experts_of_a_shard(pkg):
    """A context that holds experts [2, 6): its lists name these alone, counted from the first."""
    E, k, D, F, T, first, count = 8, 3, 256, 256, 25, 2, 4
    dims, sel, _, _, _, (hq, hs), (_, _, (d, ds)) = _experts_case(pkg, T, E, k, D, F, seed=9)
    with pkg.Context(dims, n_layer=1, max_tokens=T, device=0, expert_first=first, expert_count=count) as c:
        d_sel, = _dev(c, sel)
        d_off, d_pairs = c.alloc((count + 1) * 4), c.alloc(T * k * 4)
        c.moe_group_pairs(d_sel, T, d_off, d_pairs)
        dev = _dev(c, d[first:first + count], ds[first:first + count], hq, hs)
        d_out, = _dev(c, np.full((T, k, D), 9.5, np.float32))
        c.moe_down_grouped_fp8(*dev, d_sel, d_off, d_pairs, d_out, T)
        c.sync()
        got = d_out.download(np.float32, (T, k, D))
        _free(d_sel, d_off, d_pairs, d_out, *dev)
    for t in range(T):
        for j in range(k):
            e = sel["ids"][t, j]
            if not first <= e < first + count:
                assert np.all(got[t, j] == 9.5)
                continue
            r = t * (k + 1) + j
            wd, bd = ref.product(d[e], ds[e], hq[r:r + 1], hs[r:r + 1])
            assert np.all(np.abs(got[t, j] - sel["w"][t, j] * wd) <= bd)


def test_no_tokens_and_no_pairs(pkg):
    dims = pkg.synth.Dims(n_embd=256, n_ff=256, n_expert=4, n_used=2)
    with pkg.Context(dims, n_layer=1, max_tokens=1, device=0) as c:
        w, out = c.alloc(4 * 256 * 256), c.alloc(1 << 16)
        before = c.launch_count()
        c.moe_gateup_grouped_fp8(w, w, w, w, w, w, w, w, out, 0)
        c.moe_shared_down_fp8(w, w, w, w, w, out, 0)
        assert c.launch_count() == before
        d_off, d_out = _dev(c, np.zeros(5, np.uint32), np.full(5 * 2 * 256, 9.5, np.float32))
        c.moe_down_grouped_fp8(w, w, w, w, w, d_off, w, d_out, 5)   # a shard that none of the tokens chose
        c.sync()
        assert np.all(d_out.download(np.float32, 5 * 2 * 256) == 9.5)
        _free(w, out, d_off, d_out)


@pytest.mark.parametrize("T,E,k,D,F", [(700, 8, 4, 2048, 256), (700, 8, 4, 2048, 512), (500, 6, 4, 2048, 768), (400, 4, 4, 1280, 1280), (1500, 16, 2, 1024, 512), (60, 8, 4, 2048, 512)])
def test_experts_many_units(pkg, T, E, k, D, F):
    """Several units a block, sums of one to ten column blocks: the barriers go through many phases.  Twice: the results are the same to the bit."""
    rng = np.random.default_rng(T + F)
    dims = pkg.synth.Dims(n_embd=D, n_ff=F, n_expert=E, n_used=k)
    sel, offsets, pairs = _selection(rng, T, E, k, 0.2)
    q, s = ref.quantize(rng.standard_normal((T, D)).astype(np.float32))
    hq, hs = ref.quantize(rng.standard_normal((T * (k + 1), F)).astype(np.float32))
    (g, gs), (u, us), (d, ds) = (ref.weights(rng, *shape, mats=E) for shape in ((F, D), (F, D), (D, F)))
    h, contrib = [], []
    with pkg.Context(dims, n_layer=1, max_tokens=1, device=0) as c:
        dev = _dev(c, g, gs, u, us, q, s, offsets, pairs, d, ds, hq, hs, sel)
        for _ in range(2):
            out = _dev(c, np.full((T, k + 1, F), 9.5, np.float32), np.full((T, k, D), 9.5, np.float32))
            c.moe_gateup_grouped_fp8(*dev[:8], out[0], T)
            c.moe_down_grouped_fp8(*dev[8:12], dev[12], dev[6], dev[7], out[1], T)
            c.sync()
            h.append(out[0].download(np.float32, (T, k + 1, F)))
            contrib.append(out[1].download(np.float32, (T, k, D)))
            _free(*out)
        _free(*dev)
    assert np.array_equal(h[0], h[1]) and np.array_equal(contrib[0], contrib[1]) and np.all(h[0][:, k] == 9.5)
    for e in range(E):
        t, j = (pairs[offsets[e]:offsets[e + 1]] >> 4).astype(int), (pairs[offsets[e]:offsets[e + 1]] & 15).astype(int)
        (wg, bg), (wu, bu) = (ref.product(m[e], ms[e], q[t], s[t]) for m, ms in ((g, gs), (u, us)))
        assert np.all(np.abs(h[0][t, j] - _silu(wg) * wu) <= _swiglu_bound(wg, wu, bg, bu)), e
        r = t * (k + 1) + j
        wd, bd = ref.product(d[e], ds[e], hq[r], hs[r])
        w = sel["w"][t, j].astype(np.float64)[:, None]
        assert np.all(np.abs(contrib[0][t, j] - w * wd) <= w * bd + 2.0**-23 * np.abs(w * wd)), e
