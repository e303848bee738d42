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


# every kind of tile, rows that fill no tile, results that start on no 16 bytes, one column block and odd numbers of them, several tiles a block
TILES = [(16, 16400, 2048), (32, 50001, 272), (100, 4097, 2064), (250, 4100, 2048), (260, 4104, 1936), (64, 40001, 1040), (1000, 4100, 2048), (1030, 4101, 1040), (700, 20000, 128),
         (2100, 9000, 272), (129, 30000, 400)]


@pytest.mark.parametrize("n,M,K", SIZES + TILES)
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


@pytest.mark.parametrize("n", [1, 24, 300])
def test_gemm_beyond_32_bits(ctx, n):
    """A matrix of more than 2^32 bytes: rows at both ends and across the 4 GB line."""
    import torch
    M, K = (1 << 20) + 37, 4112
    w = torch.randint(0, 120, (M, K), dtype=torch.uint8, device="cuda")
    ws = torch.rand((ref.blocks(M), ref.blocks(K)), device="cuda")
    rng = np.random.default_rng(n)
    q, s = ref.quantize(rng.standard_normal((n, K)).astype(np.float32))
    d_q, d_s = torch.from_numpy(q).cuda(), torch.from_numpy(s).cuda()
    y = torch.empty((n, M), device="cuda")
    torch.cuda.synchronize()
    ctx.fp8_gemm(w, ws, d_q, d_s, y, M, K, n)
    ctx.sync()
    line = (1 << 32) // K // 128 * 128
    for r0 in (0, line - 128, line, (M - 1) // 128 * 128):
        rows = slice(r0, min(r0 + 128, M))
        want, bound = ref.product(w[rows].cpu().numpy(), ws[r0 // 128:r0 // 128 + 1].cpu().numpy(), q, s)
        assert np.all(np.abs(y[:, rows].cpu().numpy() - want) <= bound), r0


def test_misaligned_results_are_refused(pkg):
    dims = pkg.synth.Dims(n_embd=256, n_ff=256, n_expert=4, n_used=2)
    with pkg.Context(dims, n_layer=1, max_tokens=1, device=0) as c:
        d = c.alloc(1 << 20)
        for bad in (lambda: c.moe_gateup_grouped_fp8(d, d, d, d, d, d, d, d, d.ptr + 4, 1), lambda: c.moe_down_grouped_fp8(d, d, d, d, d, d, d, d.ptr + 8, 1),
                    lambda: c.moe_shared_gateup_fp8(d, d, d, d, d, d, d.ptr + 12, 1), lambda: c.moe_shared_down_fp8(d, d, d, d, d, d.ptr + 4, 1),
                    lambda: c.moe_gateup_grouped_fp8(d.ptr + 1, d, d, d, d, d, d, d, d, 1), lambda: c.moe_down_grouped_fp8(d, d, d.ptr + 8, d, d, d, d, d, 1),
                    lambda: c.moe_gateup_grouped_fp8(d, d, d, d, d, d, None, d, d, 1)):
            with pytest.raises(pkg.QkmError) as ei:
                bad()
            assert ei.value.code == -1
        with pytest.raises(pkg.QkmError) as ei:
            c.moe_down_grouped_fp8(d, d, d, d, d, d, d, d, 1 << 27)
        assert ei.value.code == -3
        d.free()


@pytest.mark.parametrize("T", [3, 60, 400])
def test_captured_and_replayed_on_a_stream(pkg, T):
    """The whole chain of an FP8 layer on a stream of the caller's, captured once and replayed on other inputs: the bits of the eager calls."""
    import torch
    E, k, D, F = 8, 4, 512, 512
    rng = np.random.default_rng(T)
    dims = pkg.synth.Dims(n_embd=D, n_ff=F, n_expert=E, n_used=k)
    sel, offsets, pairs = _selection(rng, T, E, k)
    mats = [t for shape in ((F, D), (F, D), (D, F)) for t in ref.weights(rng, *shape, mats=E)]
    dev = [torch.from_numpy(np.ascontiguousarray(a).view(np.uint8).reshape(-1)).cuda() for a in (*mats, sel, offsets, pairs)]
    g, gs, u, us, d, ds, d_sel, d_off, d_pairs = dev
    xs = [torch.from_numpy(rng.standard_normal((T, D)).astype(np.float32)).cuda() for _ in range(2)]
    x, logits = torch.empty_like(xs[0]), torch.randn((T, E), device="cuda")
    q, s = torch.empty((T, D), dtype=torch.uint8, device="cuda"), torch.empty((T, D // 128), device="cuda")
    hq, hs = torch.empty((T * (k + 1), F), dtype=torch.uint8, device="cuda"), torch.empty((T * (k + 1), F // 128), device="cuda")
    h, contrib = torch.zeros((T, k + 1, F), device="cuda"), torch.zeros((T, k, D), device="cuda")
    y, counts, probs, loss, grad = torch.zeros((T, F), device="cuda"), torch.zeros(E + 1, dtype=torch.int32, device="cuda"), torch.zeros(E, device="cuda"), torch.zeros(1, device="cuda"), torch.zeros((T, E), device="cuda")
    st = torch.cuda.Stream()
    with pkg.Context(dims, n_layer=1, max_tokens=1, device=0) as c:
        c.set_stream(st.cuda_stream)

        def chain():
            c.moe_balance(logits, d_sel, None, T, 0.01, counts, probs, loss)
            c.moe_balance_grad(logits, None, counts, T, 0.01, None, grad)
            c.fp8_quantize(x, T, D, q, s)
            c.fp8_gemm(g, gs, q, s, y, F, D, T)
            c.moe_gateup_grouped_fp8(g, gs, u, us, q, s, d_off, d_pairs, h, T)
            c.fp8_quantize(h, T * (k + 1), F, hq, hs)
            c.moe_down_grouped_fp8(d, ds, hq, hs, d_sel, d_off, d_pairs, contrib, T)

        outs, graph = [], torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.stream(st):
            for xi in xs:
                x.copy_(xi)
                chain()
                outs.append([t.clone() for t in (y, h, contrib, loss, counts, grad)])
            st.synchronize()
            with torch.cuda.graph(graph, stream=st):
                chain()
            for xi, want in zip(xs, outs):
                for t in (y, h, contrib, loss, counts, grad):
                    t.zero_()
                x.copy_(xi)
                graph.replay()
                for t, w in zip((y, h, contrib, loss, counts, grad), want):
                    assert torch.equal(t, w)
            st.synchronize()
        c.sync()
        del graph


def test_layer_chain(pkg):
    """The operators as a layer uses them: router logits and selection, load, pairs by expert, FP8 gate/up and down of routed and shared experts, the fold with
    the residual and the norm.  Each stage against 64 bits from what the stage before gave."""
    from qwen_kernel_b200 import SEL_DTYPE
    T, E, k, D, F = 70, 16, 4, 512, 256
    rng = np.random.default_rng(1)
    dims = pkg.synth.Dims(n_embd=D, n_ff=F, n_expert=E, n_used=k)
    x = rng.standard_normal((T, D)).astype(np.float32)
    resid = rng.standard_normal((T, D)).astype(np.float32)
    router = (rng.standard_normal((E, D)) * 0.05).astype(np.float32)
    gis, norm = (rng.standard_normal(D) * 0.05).astype(np.float32), np.ones(D, np.float32)
    routed = [ref.weights(rng, *shape, mats=E) for shape in ((F, D), (F, D), (D, F))]
    shared = [ref.weights(rng, *shape) for shape in ((F, D), (F, D), (D, F))]
    with pkg.Context(dims, n_layer=1, max_tokens=T, device=0) as c:
        d_x, d_resid, d_router, d_gis, d_norm = _dev(c, x, resid, router, gis, norm)
        d_logits, d_sel, d_off, d_pairs = c.alloc(T * E * 4), c.alloc(T * 160), c.alloc((E + 1) * 4), c.alloc(T * k * 4)
        d_counts, d_probs, d_loss = c.alloc((E + 1) * 4), c.alloc(E * 4), c.alloc(4)
        d_q, d_s, d_h = c.alloc(T * D), c.alloc(T * D // 128 * 4), c.alloc(T * (k + 1) * F * 4)
        d_hq, d_hs, d_contrib, d_y2 = c.alloc(T * (k + 1) * F), c.alloc(T * (k + 1) * F // 128 * 4), c.alloc(T * k * D * 4), c.alloc(T * D * 4)
        d_out, d_xn = c.alloc(T * D * 4), c.alloc(T * D * 4)
        (g, gs), (u, us), (d, ds) = [_dev(c, *m) for m in routed]
        (sg, sgs), (su, sus), (sd, sds) = [_dev(c, *m) for m in shared]
        c.moe_logits(0, d_router, d_x, d_logits, T)
        c.moe_select(d_logits, d_gis, d_x, d_sel, T)
        c.moe_balance(d_logits, d_sel, None, T, 1.0, d_counts, d_probs, d_loss)
        c.moe_group_pairs(d_sel, T, d_off, d_pairs)
        c.fp8_quantize(d_x, T, D, d_q, d_s)
        c.moe_gateup_grouped_fp8(g, gs, u, us, d_q, d_s, d_off, d_pairs, d_h, T)
        c.moe_shared_gateup_fp8(sg, sgs, su, sus, d_q, d_s, d_h, T)
        c.fp8_quantize(d_h, T * (k + 1), F, d_hq, d_hs)
        c.moe_down_grouped_fp8(d, ds, d_hq, d_hs, d_sel, d_off, d_pairs, d_contrib, T)
        c.moe_shared_down_fp8(sd, sds, d_hq, d_hs, d_sel, d_y2, T)
        c.add_rms3_grouped(d_resid, d_contrib, d_y2, d_norm, d_out, d_xn, T, D, k)
        c.sync()
        sel, off, counts = d_sel.download(SEL_DTYPE, T), d_off.download(np.uint32, E + 1), d_counts.download(np.uint32, E + 1)
        h, contrib = d_h.download(np.float32, (T, k + 1, F)), d_contrib.download(np.float32, (T, k, D))
        y2, out, loss = d_y2.download(np.float32, (T, D)), d_out.download(np.float32, (T, D)), d_loss.download(np.float32, 1)[0]
    assert np.array_equal(counts[:E], np.diff(off)) and counts[E] == T       # the load is what the pairs were grouped by
    logits = x.astype(np.float64) @ router.astype(np.float64).T
    p = np.exp(logits - logits.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    assert abs(loss - E / (T * k) * (counts[:E] * p.mean(0)).sum()) < 1e-4
    q, s = ref.quantize(x)
    hq, hs = ref.quantize(h.reshape(-1, F))
    for e in range(E + 1):
        t, j = np.nonzero(sel["ids"][:, :k] == e) if e < E else (np.arange(T), np.full(T, k))
        if t.size == 0:
            continue
        m = [(w[e], ws[e]) for w, ws in routed] if e < E else shared
        (wg, bg), (wu, bu) = ref.product(*m[0], q[t], s[t]), ref.product(*m[1], q[t], s[t])
        assert np.all(np.abs(h[t, j] - _silu(wg) * wu) <= _swiglu_bound(wg, wu, bg, bu)), e
        wd, bd = ref.product(*m[2], hq[t * (k + 1) + j], hs[t * (k + 1) + j])
        w = (sel["w"][t, j] if e < E else sel["w_shared"][t]).astype(np.float64)[:, None]
        got = contrib[t, j] if e < E else y2
        assert np.all(np.abs(got - w * wd) <= w * bd + 2.0**-23 * np.abs(w * wd)), e
    fold = resid.astype(np.float64) + contrib.sum(1, dtype=np.float64) + y2
    assert np.all(np.abs(out - fold) <= (k + 3) * 2.0**-23 * (np.abs(resid) + np.abs(contrib).sum(1) + np.abs(y2)))


def test_two_contexts_on_two_streams(pkg):
    """Calls of two contexts under way at the same time give what they give one after the other."""
    import torch
    E, k, D, F, T = 16, 4, 1024, 512, 600
    rng = np.random.default_rng(4)
    dims = pkg.synth.Dims(n_embd=D, n_ff=F, n_expert=E, n_used=k)
    sel, offsets, pairs = _selection(rng, T, E, k, 0.1)
    mats = [t for shape in ((F, D), (F, D), (D, F)) for t in ref.weights(rng, *shape, mats=E)]
    g, gs, u, us, d, ds, d_sel, d_off, d_pairs = [torch.from_numpy(np.ascontiguousarray(a).view(np.uint8).reshape(-1)).cuda() for a in (*mats, sel, offsets, pairs)]
    logits = torch.randn((T, E), device="cuda")
    runs = []
    for i in range(2):
        b = {"x": torch.randn((T, D), device="cuda"), "q": torch.empty((T, D), dtype=torch.uint8, device="cuda"), "s": torch.empty((T, D // 128), device="cuda"),
             "h": torch.zeros((T, k + 1, F), device="cuda"), "hq": torch.empty((T * (k + 1), F), dtype=torch.uint8, device="cuda"),
             "hs": torch.empty((T * (k + 1), F // 128), device="cuda"), "out": torch.zeros((T, k, D), device="cuda"), "y": torch.zeros((T, E * F), device="cuda"),
             "counts": torch.zeros(E + 1, dtype=torch.int32, device="cuda"), "probs": torch.zeros(E, device="cuda"), "loss": torch.zeros(1, device="cuda")}
        runs.append(b)
    streams = [torch.cuda.Stream() for _ in range(2)]
    ctxs = [pkg.Context(dims, n_layer=1, max_tokens=1, device=0) for _ in range(2)]

    def step(c, b):
        c.fp8_quantize(b["x"], T, D, b["q"], b["s"])
        c.fp8_gemm(g, gs, b["q"], b["s"], b["y"], E * F, D, T)
        c.moe_gateup_grouped_fp8(g, gs, u, us, b["q"], b["s"], d_off, d_pairs, b["h"], T)
        c.fp8_quantize(b["h"], T * (k + 1), F, b["hq"], b["hs"])
        c.moe_down_grouped_fp8(d, ds, b["hq"], b["hs"], d_sel, d_off, d_pairs, b["out"], T)
        c.moe_balance(logits, d_sel, None, T, 1.0, b["counts"], b["probs"], b["loss"])

    torch.cuda.synchronize()
    want = []
    for c, b, st in zip(ctxs, runs, streams):
        c.set_stream(st.cuda_stream)
        step(c, b)
        c.sync()
        want.append([b[n].clone() for n in ("y", "h", "out", "counts", "loss")])
    torch.cuda.synchronize()
    for _ in range(5):
        for c, b in zip(ctxs, runs):
            step(c, b)
    for c in ctxs:
        c.sync()
    for b, w in zip(runs, want):
        assert all(torch.equal(b[n], t) for n, t in zip(("y", "h", "out", "counts", "loss"), w))
    for c in ctxs:
        c.close()
