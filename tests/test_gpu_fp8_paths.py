"""FP8 products: every kernel, told by the library's own rules, so that another choice of kernel cannot leave one untested."""
import numpy as np
import pytest

import fp8_choice as choice
import fp8_ref as ref
from test_gpu_fp8 import _dev, _free, _selection, _silu, _swiglu_bound

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,F,T", [(512, 256, 1500), (1024, 512, 700), (2048, 1024, 180), (2048, 512, 330)])
def test_shared_expert_with_rows_as_lanes(pkg, D, F, T):
    """As many rows as take the kernels with the rows as lanes, down sums of two to eight column blocks; a ragged last tile."""
    k = 2
    assert not choice.shared_few_rows(False, T + 1000, F, D) and not choice.shared_few_rows(True, T, D, F)
    rng = np.random.default_rng(T)
    dims = pkg.synth.Dims(n_embd=D, n_ff=F, n_expert=4, n_used=k)
    with pkg.Context(dims, n_layer=1, max_tokens=1, device=0) as c:
        (g, gs), (u, us), (d, ds) = ref.weights(rng, F, D), ref.weights(rng, F, D), ref.weights(rng, D, F)
        for n in (T, T + 1000):
            sel, _, _ = _selection(rng, n, 4, k)
            q, s = ref.quantize(rng.standard_normal((n, D)).astype(np.float32))
            hq, hs = ref.quantize(rng.standard_normal((n * (k + 1), F)).astype(np.float32))
            dev = _dev(c, g, gs, u, us, q, s, np.full((n, k + 1, F), 9.5, np.float32))
            c.moe_shared_gateup_fp8(*dev, n)
            c.sync()
            h = dev[-1].download(np.float32, (n, k + 1, F))
            _free(*dev)
            dev = _dev(c, d, ds, hq, hs, sel, np.full((n, D), 9.5, np.float32))
            c.moe_shared_down_fp8(*dev, n)
            c.sync()
            y2 = dev[-1].download(np.float32, (n, D))
            _free(*dev)
            assert np.all(h[:, :k] == 9.5)
            (wg, bg), (wu, bu) = ref.product(g, gs, q, s), ref.product(u, us, q, s)
            assert np.all(np.abs(h[:, k] - _silu(wg) * wu) <= _swiglu_bound(wg, wu, bg, bu))
            at = np.arange(n) * (k + 1) + k
            wd, bd = ref.product(d, ds, hq[at], hs[at])
            w = sel["w_shared"].astype(np.float64)[:, None]
            assert np.all(np.abs(y2 - w * wd) <= w * bd + 2.0**-23 * np.abs(w * wd))


# rows, weight rows and columns that take each kernel; no size fills a tile, the last column block is short
PATHS = {"rows": (40, 300, 400), "group": (16, 20003, 400), "128x32": (200, 1010, 400), "128x64": (260, 2110, 400), "256x128": (300, 4110, 400), "128x256": (100, 20003, 400),
         "256x256": (520, 4110, 400)}
assert set(PATHS) == set(choice.DENSE)


@pytest.fixture(scope="module")
def ctx(pkg):
    c = pkg.Context(pkg.synth.Dims(), n_layer=1, max_tokens=16, device=0)
    yield c
    c.close()


@pytest.fixture(scope="module")
def n_sms():
    import torch
    return torch.cuda.get_device_properties(0).multi_processor_count


def _gemm(ctx, w, ws, q, s):
    M, (n, K) = w.shape[0], q.shape
    d = _dev(ctx, w, ws, q, s)
    d_y, = _dev(ctx, np.full(n * M + 64, -7.25, np.float32))
    ctx.fp8_gemm(*d, d_y, M, K, n)
    ctx.sync()
    y = d_y.download(np.float32, n * M + 64)
    _free(*d, d_y)
    assert np.all(y[n * M:] == -7.25)
    return y[:n * M].reshape(n, M)


def _by_blocks(w, ws, q, s):
    """(y, bound, sure): the definition with every block's sum scaled as a whole, so that a scale may be infinite; how far finite results may be off (fp8_ref.product);
    whether an infinite one's sign is beyond rounding."""
    W, X = ref.decode(w), ref.decode(q)
    (M, K), n = W.shape, X.shape[0]
    y, size, sure = np.zeros((n, M)), np.zeros((n, M)), np.ones((n, M), bool)
    with np.errstate(invalid="ignore", over="ignore"):
        for b in range(ref.blocks(K)):
            at = slice(128 * b, min(128 * b + 128, K))
            scale = s[:, b].astype(np.float64)[:, None] * ws[:, b].astype(np.float64).repeat(128)[:M]
            sums, sizes = X[:, at] @ W[:, at].T, np.abs(X[:, at]) @ np.abs(W[:, at]).T
            y += scale * sums
            size += np.abs(scale) * sizes
            sure &= ~np.isinf(scale) | (np.abs(sums) > sizes * 2.0**-16)
    return y, size * 2.0**-23 * (128 + ref.blocks(K) + 4), sure


def _same(got, want, bound, sure):
    infinite = np.isinf(want)
    assert sure.mean() > 0.99
    assert np.array_equal(np.isnan(got)[sure], np.isnan(want)[sure])
    assert np.array_equal(got[infinite & sure], want[infinite & sure])
    there = np.isfinite(want)
    off = np.abs(got[there] - want[there])
    assert np.all(off <= bound[there]), np.max(off / bound[there])


@pytest.mark.parametrize("path", choice.DENSE)
def test_a_spoilt_row_spoils_itself_alone(ctx, n_sms, path):
    """NaN codes in the first, a middle and the last row of either side, in the first column, a middle one and the last of the short block; scales of zero, negative and infinite
    ones.  Rows and columns of a tile that are not there, and what an earlier tile left in shared memory, reach nothing."""
    n, M, K = PATHS[path]
    assert choice.dense_kernel(n, M, K, n_sms) == path
    rng = np.random.default_rng(n)
    w, ws = ref.weights(rng, M, K)
    q, s = ref.quantize(rng.standard_normal((n, K)).astype(np.float32))
    spoilt = w.copy(), q.copy()
    for row, col in ((0, K - 1), (M // 2, 130), (M - 1, 0)):
        spoilt[0][row, col] = 127
    for row, col in ((0, 0), (n // 2, K - 1), (n - 1, 255)):
        spoilt[1][row, col] = 255
    ws[0, 1], s[n - 2, 2], ws[1, 0] = 0, 0, -0.01
    _same(_gemm(ctx, spoilt[0], ws, spoilt[1], s), *_by_blocks(spoilt[0], ws, spoilt[1], s))
    s[3, 0], ws[M // 256, 2] = np.inf, -np.inf
    _same(_gemm(ctx, w, ws, q, s), *_by_blocks(w, ws, q, s))


@pytest.mark.parametrize("path", choice.DENSE)
def test_small_products_beside_a_large_one(ctx, n_sms, path):
    """A block's sum keeps what is 2^-23 of it: 2^-9 in every column but one of 448 times 1 and 448, at the block's start, inside it and at its end."""
    n, M, K = PATHS[path]
    assert choice.dense_kernel(n, M, K, n_sms) == path
    w = np.full((M, K), ref.encode(1.0), np.uint8)
    q = np.full((n, K), 1, np.uint8)
    for b, at in enumerate((0, 128 + 77, 256 + 127, K - 1)):
        q[:, at] = 126 if b % 2 else 254
        w[1::2, at] = 126
    ones = np.ones((ref.blocks(M), ref.blocks(K)), np.float32), np.ones((n, ref.blocks(K)), np.float32)
    _same(_gemm(ctx, w, ones[0], q, ones[1]), *_by_blocks(w, ones[0], q, ones[1]))


@pytest.mark.parametrize("path", choice.DENSE)
def test_blocks_that_cancel(ctx, n_sms, path):
    """Two blocks 2^30 above the others, one the other's opposite: what f32 sums keep of the rest stays."""
    n, M, K = PATHS[path]
    assert choice.dense_kernel(n, M, K, n_sms) == path
    rng = np.random.default_rng(M)
    w, ws = ref.weights(rng, M, K)
    q, s = ref.quantize(rng.standard_normal((n, K)).astype(np.float32))
    w[:, 128:256] = w[:, :128]
    q[:, 128:256] = q[:, :128] ^ 128
    s[:, 1] = s[:, 0]
    ws[:, 0] = ws[:, 1] = 2.0**20
    _same(_gemm(ctx, w, ws, q, s), *_by_blocks(w, ws, q, s))


# tokens, experts, selections, hidden, inner: gate/up and down by columns, by lanes (down of few column blocks and of more)
EXPERT_PATHS = [(20, 4, 2, 256, 256), (300, 4, 2, 512, 256), (300, 4, 2, 256, 768)]


@pytest.mark.parametrize("T,E,k,D,F", EXPERT_PATHS)
def test_a_spoilt_pair_spoils_itself_alone(pkg, T, E, k, D, F):
    """NaN codes in one weight row of an expert and in single tokens' rows, zero, negative and infinite scales, a large product beside small ones: every other result of
    gate/up and down is as without them."""
    lanes = T == 300
    assert choice.pairs_as_lanes(False, T, k, E) == choice.pairs_as_lanes(True, T, k, E) == lanes
    rng = np.random.default_rng(T + F)
    dims = pkg.synth.Dims(n_embd=D, n_ff=F, n_expert=E, n_used=k)
    sel, offsets, pairs = _selection(rng, T, E, k)
    q, s = ref.quantize(rng.standard_normal((T, D)).astype(np.float32))
    hq, hs = ref.quantize(rng.standard_normal((T * (k + 1), F)).astype(np.float32))
    (g, gs), (u, us), (d, ds) = (ref.weights(rng, *shape, mats=E) for shape in ((F, D), (F, D), (D, F)))
    g[1, 0, D - 1], u[2, F - 1, 0], d[1, D // 2, 130], d[3, D - 1, F - 1] = 127, 255, 127, 255
    q[T - 1, D - 1], hq[0, 0], hq[(T // 2) * (k + 1) + 1, F - 1] = 127, 255, 127
    gs[0, 1, 0], us[3, 0, 1], ds[0, 0, 1], ds[2, 1, 0] = -0.01, 0, 0, np.inf
    s[2, 1], hs[4 * (k + 1), 0] = 0, np.inf
    q[5], q[5, 200] = 1, 126
    hq[6 * (k + 1)], hq[6 * (k + 1), 3] = 1, 254
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
    for e in range(E):
        p = pairs[offsets[e]:offsets[e + 1]]
        t, j = (p >> 4).astype(int), (p & 15).astype(int)
        (wg, bg, _), (wu, bu, _) = _by_blocks(g[e], gs[e], q[t], s[t]), _by_blocks(u[e], us[e], q[t], s[t])
        want = _silu(wg) * wu
        assert np.array_equal(np.isnan(h[t, j]), np.isnan(want)), e
        there = ~np.isnan(want)
        assert np.all(np.abs(h[t, j] - want)[there] <= _swiglu_bound(wg, wu, bg, bu)[there]), e
        r = t * (k + 1) + j
        wd, bd, sure = _by_blocks(d[e], ds[e], hq[r], hs[r])
        w = sel["w"][t, j].astype(np.float64)[:, None]
        _same(contrib[t, j], w * wd, w * bd + 2.0**-23 * np.abs(w * wd), sure)


def _run_gateup_down(c, T, k, D, F, mats, q, s, hq, hs, d_sel, d_off, d_pairs):
    (g, gs), (u, us), (d, ds) = mats
    dev = _dev(c, g, gs, u, us, q, s, d, ds, hq, hs, np.full((T, k + 1, F), 9.5, np.float32), np.full((T, k, D), 9.5, np.float32))
    c.moe_gateup_grouped_fp8(*dev[:6], d_off, d_pairs, dev[10], T)
    c.moe_down_grouped_fp8(*dev[6:10], d_sel, d_off, d_pairs, dev[11], T)
    c.sync()
    got = dev[10].download(np.float32, (T, k + 1, F)), dev[11].download(np.float32, (T, k, D))
    _free(*dev)
    return got


def _check_pairs(mats, q, s, hq, hs, sel, h, contrib, k, of_expert):
    """Every slot against 64 bits; of_expert: {expert's place in mats: (tokens, slots)}; all other slots hold 9.5."""
    (g, gs), (u, us), (d, ds) = mats
    held = np.ones(h.shape[:2], bool)
    for e, (t, j) in of_expert.items():
        held[t, j] = False
        (wg, bg), (wu, bu) = (ref.product(m[e], ms[e], q[t], s[t]) for m, ms in ((g, gs), (u, us)))
        assert np.all(np.abs(h[t, j] - _silu(wg) * wu) <= _swiglu_bound(wg, wu, bg, bu)), e
        r = t * (k + 1) + j
        wd, bd = ref.product(d[e], ds[e], hq[r], hs[r])
        w = sel["w"][t, j].astype(np.float64)[:, None]
        assert np.all(np.abs(contrib[t, j] - w * wd) <= w * bd + 2.0**-23 * np.abs(w * wd)), e
    assert np.all(h[held] == 9.5) and np.all(contrib[held[:, :k]] == 9.5)


def _case(rng, T, E, k, D, F):
    mats = [ref.weights(rng, *shape, mats=E) for shape in ((F, D), (F, D), (D, F))]
    return mats, *ref.quantize(rng.standard_normal((T, D)).astype(np.float32)), *ref.quantize(rng.standard_normal((T * (k + 1), F)).astype(np.float32))


@pytest.mark.parametrize("T,F", [(7, 256), (130, 256), (130, 768)])
def test_gateup_and_down_of_lists_with_strangers(pkg, T, F):
    """Pairs that name a token or a slot that there is none of, an expert whose run ends before it begins, an offset past the list: the rest is computed, nothing else written."""
    E, k, D = 4, 2, 256
    assert choice.pairs_as_lanes(False, T, k, E) == choice.pairs_as_lanes(True, T, k, E) == (T == 130)
    rng = np.random.default_rng(T + F)
    dims = pkg.synth.Dims(n_embd=D, n_ff=F, n_expert=E, n_used=k)
    sel, offsets, pairs = _selection(rng, T, E, k)
    mats, q, s, hq, hs = _case(rng, T, E, k, D, F)
    good = np.ones(pairs.size, bool)
    for i, v in ((0, T << 4), (3, 0xFFFFFFF0), (5, 0 << 4 | k), (offsets[3], 0xFFFFFFFF), (pairs.size - 1, 15)):
        pairs[i], good[i] = v, False
    offsets[2] = offsets[1] - 1                                # expert 1's run ends before it begins; expert 2 has its pairs and the last of expert 0
    offsets[4] += 1000
    of_expert = {}
    for e in (0, 2, 3):
        p = np.arange(offsets[e], min(offsets[e + 1], pairs.size))
        if e == 0:
            p = p[:-1]                                         # (that one pair is written by both)
        p = pairs[p[good[p]]]
        of_expert[e] = (p >> 4).astype(int), (p & 15).astype(int)
    both = pairs[offsets[1] - 1]
    with pkg.Context(dims, n_layer=1, max_tokens=1, device=0) as c:
        dev = _dev(c, sel, offsets, pairs)
        h, contrib = _run_gateup_down(c, T, k, D, F, mats, q, s, hq, hs, *dev)
        _free(*dev)
    if good[offsets[1] - 1]:
        t, j = int(both >> 4), int(both & 15)
        of_expert[2] = tuple(np.delete(a, np.flatnonzero((of_expert[2][0] == t) & (of_expert[2][1] == j))) for a in of_expert[2])
        assert not np.all(h[t, j] == 9.5)
        h[t, j], contrib[t, j] = 9.5, 9.5
    _check_pairs(mats, q, s, hq, hs, sel, h, contrib, k, of_expert)


@pytest.mark.parametrize("T,F", [(25, 256), (300, 256), (300, 768)])
def test_gateup_and_down_of_a_shard(pkg, T, F):
    """A context that holds experts [2, 6) of 8: lists count from the first of them, pairs of the others are not there."""
    E, k, D, first, count = 8, 3, 256, 2, 4
    assert choice.pairs_as_lanes(False, T, k, E) == choice.pairs_as_lanes(True, T, k, E) == (T == 300)
    rng = np.random.default_rng(T + F)
    dims = pkg.synth.Dims(n_embd=D, n_ff=F, n_expert=E, n_used=k)
    sel, _, _ = _selection(rng, T, E, k)
    mats, q, s, hq, hs = _case(rng, T, count, k, D, F)
    with pkg.Context(dims, n_layer=1, max_tokens=T, device=0, expert_first=first, expert_count=count) as c:
        d_sel, = _dev(c, sel)
        d_off, d_pairs = c.alloc((count + 1) * 4), c.alloc(T * k * 4)
        c.moe_group_pairs(d_sel, T, d_off, d_pairs)
        h, contrib = _run_gateup_down(c, T, k, D, F, mats, q, s, hq, hs, d_sel, d_off, d_pairs)
        _free(d_sel, d_off, d_pairs)
    _check_pairs(mats, q, s, hq, hs, sel, h, contrib, k, {e: np.nonzero(sel["ids"][:, :k] == first + e) for e in range(count)})


def test_two_contexts_at_a_time_write_everything(pkg):
    """Two contexts' layers on two streams, other inputs every round, every result and everything between spoilt ahead of each: the bits of the calls one after the other."""
    import torch
    E, k, D, F, T = 16, 4, 1024, 512, 600
    assert choice.pairs_as_lanes(True, T, k, E)
    rng = np.random.default_rng(6)
    dims = pkg.synth.Dims(n_embd=D, n_ff=F, n_expert=E, n_used=k)
    sel, offsets, pairs = _selection(rng, T, E, k, 0.1)
    mats = [t for shape in ((F, D), (F, D), (D, F)) for t in ref.weights(rng, *shape, mats=E)]
    g, gs, u, us, d, ds, d_sel, d_off, d_pairs = [torch.from_numpy(np.ascontiguousarray(a).view(np.uint8).reshape(-1)).cuda() for a in (*mats, sel, offsets, pairs)]
    xs, logits = [torch.randn((T, D), device="cuda") for _ in range(3)], [torch.randn((T, E), device="cuda") for _ in range(3)]
    empty = {"q": ((T, D), torch.uint8), "s": ((T, D // 128), torch.float32), "h": ((T, k + 1, F), torch.float32), "hq": ((T * (k + 1), F), torch.uint8),
             "hs": ((T * (k + 1), F // 128), torch.float32), "out": ((T, k, D), torch.float32), "y": ((T, E * F), torch.float32), "y2": ((T, D), torch.float32),
             "counts": ((E + 1,), torch.int32), "probs": ((E,), torch.float32), "loss": ((1,), torch.float32), "grad": ((T, E), torch.float32)}
    runs = [{n: torch.empty(shape, dtype=t, device="cuda") for n, (shape, t) in empty.items()} for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    ctxs = [pkg.Context(dims, n_layer=1, max_tokens=1, device=0) for _ in range(2)]
    results = ("q", "s", "h", "hq", "hs", "out", "y", "y2", "counts", "probs", "loss", "grad")

    def step(c, b, i):
        for t in b.values():
            t.fill_(float("nan") if t.dtype == torch.float32 else 0x5A)
        c.fp8_quantize(xs[i], T, D, b["q"], b["s"])
        c.fp8_gemm(g, gs, b["q"], b["s"], b["y"], E * F, D, T)
        c.moe_gateup_grouped_fp8(g, gs, u, us, b["q"], b["s"], d_off, d_pairs, b["h"], T)
        c.moe_shared_gateup_fp8(g, gs, u, us, b["q"], b["s"], b["h"], T)
        c.fp8_quantize(b["h"], T * (k + 1), F, b["hq"], b["hs"])
        c.moe_down_grouped_fp8(d, ds, b["hq"], b["hs"], d_sel, d_off, d_pairs, b["out"], T)
        c.moe_shared_down_fp8(d, ds, b["hq"], b["hs"], d_sel, b["y2"], T)
        c.moe_balance(logits[i], d_sel, None, T, 1.0, b["counts"], b["probs"], b["loss"])
        c.moe_balance_grad(logits[i], None, b["counts"], T, 1.0, None, b["grad"])
        return [b[n].clone() for n in results]

    for c, st in zip(ctxs, streams):
        c.set_stream(st.cuda_stream)
    torch.cuda.synchronize()
    want = []
    for i in range(3):
        with torch.cuda.stream(streams[0]):
            want.append(step(ctxs[0], runs[0], i))
        torch.cuda.synchronize()
    for w in want:
        assert not any(torch.isnan(t).any() for t in w if t.dtype == torch.float32)
    got = []
    for r in range(9):
        for x, (c, b, st) in enumerate(zip(ctxs, runs, streams)):
            with torch.cuda.stream(st):
                got.append(((r + x) % 3, step(c, b, (r + x) % 3)))
    torch.cuda.synchronize()
    for c in ctxs:
        c.sync()
        c.close()
    for i, outs in got:
        for name, a, w in zip(results, outs, want[i]):
            assert torch.equal(a, w), name
