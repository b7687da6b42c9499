"""The short causal convolution and the selective state space scan in the cases
at their borders; the formulas in 64 bits and the tolerances are test_sequence_ops'."""
import math

import pytest
import torch

from dlvk_b200.ops import ssm
from test_sequence_ops import DEVICES, DTYPES, limits, near, run_scan, run_scan_bwd, scan_check, scan_inputs, scan_ref


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,N,G", [(1, 16, 1), (5, 16, 1), (23, 5, 1), (300, 16, 1), (40, 33, 2)])
def test_scan_of_rates_past_fp32(device, dtype, T, N, G):
    """exp(a_log) past fp32's largest value: a token of any length leaves nothing
    of the state, one of no length (masked, or behind its sequence) all of it.
    Decays of 0 have no error, so the tolerance is that of the other states."""
    p, dy, state, _ = scan_inputs(3, T, 24, N, G, dtype, device, T + N)
    p["dt"], p["dt_bias"] = p["dt"].clamp(-4, 4), p["dt_bias"].clamp(-4, 4)  # steps of 3e-4 and more
    p["a_log"] = p["a_log"].clamp(max=2.0)
    xmax = scan_ref(p, None, state, None)[3]
    p["a_log"][3:9] = 90.0
    p["a_log"][10, 0] = 500.0
    p["a_log"][11, 0] = math.inf
    short, long = limits(p, xmax)
    ref = dict(p, a_log=p["a_log"].clamp(max=600.0))  # (whose rates are finite in 64 bits)
    for n in (None, torch.tensor([T, T // 2, 0], dtype=torch.int32, device=device)):
        (y, h, g, _), (my, mh, mg, _) = (scan_ref(ref, dy, state, n, absolute=a) for a in (False, True))
        gy, gh, saved = run_scan(p, state=state, lengths=n, want_state=True, save=True)
        near(gy, y, my, short, "y")
        near(gh, h, mh, short, "state")
        grads = run_scan_bwd(p, dy, saved, lengths=n)
        for k in ("u", "dt", "a_log", "b", "c", "skip", "z", "dt_bias"):
            near(getattr(grads, "d" + k), g[k], mg[k], long, k)
    masked = dict(p, dt=torch.full_like(p["dt"], -math.inf))
    y, h, saved = run_scan(masked, state=state, want_state=True, save=True)
    assert torch.equal(h, state) and bool(torch.isfinite(y).all())
    assert all(bool(torch.isfinite(v).all()) for v in run_scan_bwd(masked, dy, saved))
    nan = dict(p, a_log=p["a_log"].clone())
    nan["a_log"][5] = math.nan
    y = run_scan(nan, state=state)[0]
    assert bool(torch.isnan(y[..., 5]).all()) and bool(torch.isfinite(y[..., 6:]).all())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("G", [1, 3])
def test_scan_of_no_channels(device, dtype, G):
    """No channel reads b and c: their gradients are zeros, whatever was there."""
    p, dy, state, _ = scan_inputs(2, 19, 0, 5, G, dtype, device)
    y, last, saved = run_scan(p, state=state, want_state=True, save=True)
    assert y.shape == (2, 19, 0) and last.shape == (2, 0, 5)
    given = {k: torch.full_like(p["b"], 7.0) for k in ("db", "dc")}
    grads = run_scan_bwd(p, dy, saved, **given)
    assert not given["db"].any() and not given["dc"].any() and grads.da_log.shape == (0, 5)
