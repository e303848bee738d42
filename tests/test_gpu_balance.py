"""The router's balance loss, its counts and its gradient against 64 bits."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
FLOOR = -3.4e38


@pytest.fixture(scope="module")
def contexts(pkg):
    made = {}

    def get(E, k):
        if (E, k) not in made:
            made[E, k] = pkg.Context(pkg.synth.Dims(n_embd=256, n_ff=256, n_expert=E, n_used=k), n_layer=1, max_tokens=1, device=0)
        return made[E, k]
    yield get
    for c in made.values():
        c.close()


def _reference(logits, ids, mask, coef, d_loss):
    T, E = logits.shape
    k = ids.shape[1]
    keep = np.ones(T, bool) if mask is None else mask != 0
    fine = np.isfinite(logits)
    z = np.where(fine, logits, FLOOR).astype(np.float64)
    p = np.exp(z - z.max(1, keepdims=True)) if T else z
    p = p / p.sum(1, keepdims=True)
    N = int(keep.sum())
    chosen = ids[keep].reshape(-1)
    counts = np.bincount(chosen[chosen < E], minlength=E)
    probs = p[keep].sum(0) / max(N, 1)
    loss = coef * E / (max(N, 1) * k) * (counts * probs).sum()
    g = d_loss * coef * E / (max(N, 1) ** 2 * k) * counts
    grad = np.zeros((T, E))
    grad[keep] = p[keep] * (g - (p[keep] @ g)[:, None])
    grad[~fine] = 0
    return counts, N, probs, loss, grad, (p * (g + (p @ g)[:, None])) if T else grad


def _run(c, logits, sel, mask, coef, d_loss, in_place=False, offset=0):
    T, E = logits.shape
    raw = np.zeros(T * E + offset, np.float32)
    raw[offset:] = logits.reshape(-1)
    d_raw, d_sel = c.to_device(raw), c.to_device(sel)
    d_logits = d_raw.ptr + 4 * offset
    d_mask = None if mask is None else c.to_device(mask)
    d_counts, d_probs, d_loss_out = c.alloc((E + 1) * 4), c.alloc(E * 4), c.alloc(4)
    d_up = None if d_loss is None else c.to_device(np.array([d_loss], np.float32))
    c.moe_balance(d_logits, d_sel, d_mask, T, coef, d_counts, d_probs, d_loss_out)
    d_grad = d_raw if in_place else c.alloc((T * E + 1) * 4)
    c.moe_balance_grad(d_logits, d_mask, d_counts, T, coef, d_up, d_logits if in_place else d_grad)
    c.sync()
    counts, probs, loss = d_counts.download(np.uint32, E + 1), d_probs.download(np.float32, E), d_loss_out.download(np.float32, 1)[0]
    grad = d_grad.download(np.float32, T * E + (offset if in_place else 0))[offset if in_place else 0:].reshape(T, E)
    for b in (d_raw, d_sel, d_mask, d_counts, d_probs, d_loss_out, d_up, None if in_place else d_grad):
        if b is not None:
            b.free()
    return counts, probs, loss, grad


def _records(rng, T, E, k):
    from qwen_kernel_b200 import SEL_DTYPE
    sel = np.zeros(T, SEL_DTYPE)
    sel["ids"] = 0xFFFFFFFF                                   # what lies behind the selected ones is not looked at
    for t in range(T):
        sel["ids"][t, :k] = rng.permutation(E)[:k]
    return sel


def _check(got, want, T, E):
    """Tolerances.  A probability carries expf (2 ulp), the sum of E terms (E/32 + 5 additions, half an ulp each), the reciprocal and a product: below
    (E/32 + 12) * 2^-24 of itself.  Means: a lane adds up T / (8 * blocks) <= T of them in f32 and the rest in 64 bits.  The gradient subtracts the
    row's mean of g from g, both of which carry that error, E/32 + 5 additions and three roundings more: (E/16 + 32) * 2^-24 of p * (g + mean)."""
    counts, probs, loss, grad = got
    w_counts, N, w_probs, w_loss, w_grad, size = want
    assert np.array_equal(counts[:E], w_counts) and counts[E] == N
    rel = (E / 32 + 12 + min(T, 64)) * 2.0**-24
    assert np.all(np.abs(probs - w_probs) <= rel * w_probs + 2.0**-38 * 300)
    assert abs(loss - w_loss) <= rel * abs(w_loss) + 1e-30
    assert np.all(np.abs(grad - w_grad) <= (E / 16 + 32) * 2.0**-24 * np.abs(size) + 1e-37)


@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 256, 8), (3, 7, 2), (9, 60, 4), (64, 130, 6), (77, 512, 10), (500, 256, 8), (1000, 511, 16), (2500, 128, 8), (20000, 256, 8)])
@pytest.mark.parametrize("masked", [False, True])
def test_balance(contexts, T, E, k, masked):
    rng = np.random.default_rng(T * 1000 + E)
    logits = (rng.standard_normal((T, E)) * 3).astype(np.float32)
    sel = _records(rng, T, E, k)
    mask = (rng.random(T) < 0.6).astype(np.uint8) * 3 if masked else None
    got = _run(contexts(E, k), logits, sel, mask, 0.01, 1.5)
    _check(got, _reference(logits, sel["ids"][:, :k], mask, 0.01, 1.5), T, E)
    again = _run(contexts(E, k), logits, sel, mask, 0.01, 1.5)      # the sums in progress were left at zero, and the order of blocks does not matter
    assert all(np.array_equal(a, b) for a, b in zip(got, again))


def test_balance_masks_and_extremes(contexts):
    """Infinities, NaN, the type's lowest value, rows of nothing else; every token masked; ids past the table; the same id twice."""
    E, k, T = 64, 4, 12
    rng = np.random.default_rng(2)
    logits = rng.standard_normal((T, E)).astype(np.float32)
    logits[0, 5:20] = -np.inf
    logits[1, 3], logits[1, 4] = np.nan, np.inf
    logits[2, :] = -np.inf
    logits[3, :] = np.nan
    logits[4, :63] = np.finfo(np.float32).min
    logits[5, :] = np.finfo(np.float32).min
    logits[6, 7] = np.finfo(np.float32).max
    logits[7, :] *= 100
    sel = _records(rng, T, E, k)
    sel["ids"][8, 1] = sel["ids"][8, 0]
    sel["ids"][9, :2] = [E, 0xFFFFFFFF]
    for mask in (None, np.array([1, 0] * 6, np.uint8), np.zeros(T, np.uint8)):
        _check(_run(contexts(E, k), logits, sel, mask, 1.0, None), _reference(logits, sel["ids"][:, :k], mask, 1.0, 1.0), T, E)


@pytest.mark.parametrize("E,k,offset", [(256, 8, 0), (256, 8, 1), (255, 5, 3)])
def test_balance_in_place_and_unaligned(contexts, E, k, offset):
    T = 40
    rng = np.random.default_rng(offset)
    logits = rng.standard_normal((T, E)).astype(np.float32)
    sel = _records(rng, T, E, k)
    _check(_run(contexts(E, k), logits, sel, None, 0.1, -2.0, in_place=True, offset=offset), _reference(logits, sel["ids"][:, :k], None, 0.1, -2.0), T, E)


def test_gradient_is_the_difference_quotient(contexts):
    """The gradient against central differences of the 64-bit loss with the counts held: their error is h^2 / 6 of the third derivative, below
    h^2 * coef * E here, and 2^-50 / h of the loss."""
    T, E, k, coef, h = 6, 32, 4, 0.5, 1e-4
    rng = np.random.default_rng(11)
    logits = rng.standard_normal((T, E)).astype(np.float32)
    sel = _records(rng, T, E, k)
    counts, probs, loss, grad = _run(contexts(E, k), logits, sel, None, coef, None)

    def value(z):
        p = np.exp(z - z.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
        return coef * E / (T * k) * (counts[:E] * p.mean(0)).sum()

    z = logits.astype(np.float64)
    for t, e in ((0, 0), (0, 31), (3, 7), (5, 16)):
        up, down = z.copy(), z.copy()
        up[t, e] += h
        down[t, e] -= h
        assert abs(grad[t, e] - (value(up) - value(down)) / (2 * h)) <= h * h * coef * E + 1e-6 * np.abs(grad).max() + 1e-11


def test_balance_of_nothing_and_refusals(contexts, pkg):
    c = contexts(16, 2)
    d = c.alloc(4096)
    d_counts, d_probs, d_loss = c.to_device(np.full(17, 7, np.uint32)), c.to_device(np.full(16, 7, np.float32)), c.to_device(np.full(1, 7, np.float32))
    c.moe_balance(d, d, None, 0, 1.0, d_counts, d_probs, d_loss)
    c.moe_balance_grad(d, None, d_counts, 0, 1.0, None, d)
    c.sync()
    assert not d_counts.download(np.uint32, 17).any() and not d_probs.download(np.float32, 16).any() and d_loss.download(np.float32, 1)[0] == 0
    for bad, code in ((lambda: c.moe_balance(None, d, None, 1, 1.0, d, d, d), -1), (lambda: c.moe_balance(d, d, None, 1, 1.0, d, d, None), -1),
                      (lambda: c.moe_balance_grad(d, None, None, 1, 1.0, None, d), -1), (lambda: c.moe_balance(d, d, None, (1 << 24) + 1, 1.0, d, d, d), -3),
                      (lambda: c.moe_balance_grad(d, None, d, (1 << 24) + 1, 1.0, None, d), -3)):
        with pytest.raises(pkg.QkmError) as ei:
            bad()
        assert ei.value.code == code
    for b in (d, d_counts, d_probs, d_loss):
        b.free()


@pytest.mark.parametrize("T,E,k,kept", [(1, 64, 4, 1), (1, 512, 10, 1), (3, 60, 4, 2), (40, 256, 8, 3), (3000, 128, 8, 5)])
def test_small_probabilities_of_few_tokens(contexts, T, E, k, kept):
    """Probabilities down to e^-24 of the largest; logits are multiples of 2^-10, so their distances from the largest are exact.  Of itself a mean carries what _check counts, and beside that 2^-63 of the power of two above T (the
    rounding of its sum, an integer of 2^-62 of that power, once for each block that has a token, so at most once a token)."""
    rng = np.random.default_rng(T + E)
    logits = (np.round(rng.uniform(-24, 0, (T, E)) * 1024) / 1024).astype(np.float32)
    sel = _records(rng, T, E, k)
    mask = np.zeros(T, np.uint8)
    mask[rng.permutation(T)[:kept]] = 1
    counts, probs, loss, _ = _run(contexts(E, k), logits, sel, mask, 1.0, None)
    w_counts, N, w_probs, w_loss, _, _ = _reference(logits, sel["ids"][:, :k], mask, 1.0, 1.0)
    assert N == kept and counts[E] == kept and np.array_equal(counts[:E], w_counts)
    rel, least = (E / 32 + 12 + min(kept, 64)) * 2.0**-24, 2.0**-63 * 2 ** int(np.ceil(np.log2(T)))
    assert np.all(np.abs(probs - w_probs) <= rel * w_probs + least), np.max(np.abs(probs - w_probs) / w_probs)
    assert abs(loss - w_loss) <= rel * w_loss + least * E


@pytest.mark.parametrize("E,k", [(64, 4), (61, 3), (300, 8)])
@pytest.mark.parametrize("upstream", [np.inf, -np.inf, np.nan, 3e38])
def test_gradient_where_the_upstream_is_not_finite(contexts, E, k, upstream):
    """A loss scale that overflowed: tokens that the mask leaves out and logits that are not finite get zero all the same, the rest nothing
    finite.  (3e38 times a coefficient of 100 passes f32 too.)"""
    T = 20
    rng = np.random.default_rng(E)
    logits = rng.standard_normal((T, E)).astype(np.float32)
    logits[0, 5:20], logits[1, 3], logits[2, 4], logits[3, :], logits[4, :E - 1] = -np.inf, np.nan, np.inf, -np.inf, np.nan
    sel = _records(rng, T, E, k)
    sel["ids"][:, 0], sel["ids"][:, 1:k] = 7, 9
    mask = np.ones(T, np.uint8)
    mask[10:14] = 0
    grad = _run(contexts(E, k), logits, sel, mask, 100.0, upstream)[3]
    zero = ~np.isfinite(logits) | (mask == 0)[:, None]
    assert np.all(grad[zero] == 0) and not np.isfinite(grad[~zero]).any()


def test_calls_that_overlapped_leave_nothing_behind(contexts):
    """Two streams' calls of one context at the same time get each other's sums, as the header says; the calls after them do not."""
    import torch
    E, k = 256, 8
    c = contexts(E, k)
    rng = np.random.default_rng(1)
    parts = []
    for T in (2000, 700):
        logits, sel = rng.standard_normal((T, E)).astype(np.float32), _records(rng, T, E, k)
        parts.append((T, logits, sel, torch.from_numpy(logits).cuda(), torch.from_numpy(sel.view(np.uint8).reshape(T, -1)).cuda(),
                      torch.zeros(E + 1, dtype=torch.int32, device="cuda"), torch.zeros(E, device="cuda"), torch.zeros(1, device="cuda"), torch.cuda.Stream()))
    torch.cuda.synchronize()
    try:
        for _ in range(200):
            for T, _, _, d_logits, d_sel, counts, probs, loss, st in parts:
                c.set_stream(st.cuda_stream)
                c.moe_balance(d_logits, d_sel, None, T, 0.01, counts, probs, loss)
        torch.cuda.synchronize()
    finally:
        c.set_stream(0)
    for _ in range(2):
        for T, logits, sel, *_ in parts:
            _check(_run(c, logits, sel, None, 0.01, 1.5), _reference(logits, sel["ids"][:, :k], None, 0.01, 1.5), T, E)


def test_exponential_over_its_range(contexts):
    """The gradient of a row of two logits, 0 and -x, where the first expert has every selection: -p0 p1 g, p0 / p1 = e^-x, for x from 0 to the end of the normal numbers.  In halves of
    an ulp (2^-24 of the value): the exponential 3, as its comment says; the sum of the two 1 and what of the exponential's 3 is in it; its reciprocal 4 (__fdividef); so 12 for p0 and 9 for
    p1, with the product that makes either; one each for g, p1 g, their difference from zero's and the last product: 25, and what f32 cannot hold, 2^-126."""
    E, k, T = 2, 1, 1 << 16
    rng = np.random.default_rng(3)
    x = np.concatenate([np.linspace(0, 87.3, T - 4096), rng.uniform(0, 1, 2048) * 2.0 ** rng.integers(-20, 0, 2048), np.arange(1, 2049) / 2048 * 87]).astype(np.float32)
    logits = np.stack([-x, np.zeros_like(x)], 1)
    sel = _records(rng, T, E, k)
    sel["ids"][:, 0] = 1
    _, _, _, grad = _run(contexts(E, k), logits, sel, None, float(T), None)
    e = np.exp(-x.astype(np.float64))
    want = -e / (1 + e) ** 2 * 2.0                             # coef * E / (N^2 k) * counts = T * 2 / T^2 * T
    off = np.abs(grad[:, 0] - want)
    assert np.all(off <= 25 * 2.0**-24 * np.abs(want) + 2.0**-125), np.max((off - 2.0**-125) / np.abs(want)) * 2**24
