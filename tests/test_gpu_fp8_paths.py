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
