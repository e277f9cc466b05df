"""The rates of scaled contexts against their formulas, and the refusals of the rotation's C entry points
(made before anything is launched, so they need no device)."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

import _mtpk
import rotary


def test_plain_linear_and_ntk_rates() -> None:
    plain, m = rotary.frequencies(64, 1e4)
    want = [1e4 ** (-2 * i / 64) for i in range(32)]
    assert m == 1.0 and plain.dtype == torch.float64
    torch.testing.assert_close(plain, torch.tensor(want, dtype=torch.float64), rtol=1e-14, atol=0)
    linear, m = rotary.frequencies(64, 1e4, scaling="linear", factor=8.0)
    assert m == 1.0 and torch.equal(linear, plain / 8.0)
    ntk, _ = rotary.frequencies(64, 1e4, scaling="ntk", factor=8.0)
    assert ntk[0] == 1.0  # the fastest pair stays, the slowest is slowed by the factor
    assert math.isclose(float(ntk[-1]), float(plain[-1]) / 8.0, rel_tol=1e-13)


def test_yarn_rates() -> None:
    dim, theta, factor, original = 128, 1e6, 16.0, 4096
    plain, _ = rotary.frequencies(dim, theta)
    rates, m = rotary.frequencies(dim, theta, scaling="yarn", factor=factor, original=original)
    assert math.isclose(m, 0.1 * math.log(16.0) + 1.0)
    turns = original * plain / (2 * math.pi)
    ratio = rates / plain
    assert torch.all((ratio >= 1 / factor - 1e-15) & (ratio <= 1.0)) and torch.all(ratio[1:] <= ratio[:-1])
    # the border pairs by index are rounded outwards, so a pair next to one may be ramped a little
    assert torch.all(ratio[turns > 64] == 1.0) and torch.all((ratio[turns < 0.5] - 1 / factor).abs() < 1e-12)
    low = math.floor(dim / 2 * math.log(original / (2 * math.pi * 32)) / math.log(theta))
    high = math.ceil(dim / 2 * math.log(original / (2 * math.pi)) / math.log(theta))
    i = (low + high) // 2
    g = (i - low) / (high - low)
    assert math.isclose(float(rates[i]), float(plain[i]) * (g / factor + 1 - g), rel_tol=1e-13)


@pytest.mark.parametrize("kw", [
    {"dim": 63}, {"dim": 0}, {"theta": 0.0}, {"scaling": "other"}, {"scaling": "linear", "factor": 0.5},
    {"scaling": "yarn", "factor": 4.0}, {"scaling": "yarn", "original": 4096, "fast": 1.0},
    {"dim": 2, "scaling": "ntk", "factor": 2.0},
])  # fmt: skip
def test_frequencies_refuse(kw) -> None:
    args = {"dim": 64, "theta": 1e4, **kw}
    with pytest.raises(ValueError):
        rotary.frequencies(args.pop("dim"), args.pop("theta"), **args)


@pytest.fixture(scope="module")
def lib():
    if not _mtpk.LIB_PATH.exists():
        import __graft_entry__

        __graft_entry__.build()
    return _mtpk.lib()


P = 1 << 20  # an address that no refused call follows


def _arr(*v):
    return (ctypes.c_int64 * len(v))(*v)


ROTATE = dict(x=P, dtype=1, xs=(512, 64), tokens=4, heads=8, dim=64, w=None, w_dt=0, eps=1e-6, pos=P, rates=P, rot=64,
              inter=0, mag=1.0, out=P, os=(512, 64))


@pytest.mark.parametrize("bad", [
    {"x": None}, {"x": P + 8}, {"out": P + 2}, {"pos": None}, {"rates": None}, {"dtype": 2}, {"w": P, "w_dt": 3},
    {"dim": 60}, {"dim": 520}, {"rot": 66}, {"rot": 3}, {"rot": 0}, {"heads": 0}, {"tokens": -1}, {"xs": (512, 60)},
    {"os": (508, 64)}, {"eps": -1.0}, {"eps": float("nan")},
])  # fmt: skip
def test_rotate_refuses(lib, bad) -> None:
    a = {**ROTATE, **bad}
    xs, os_ = _arr(*a["xs"]), _arr(*a["os"])
    assert lib.mtpk_rotate(a["x"], a["dtype"], ctypes.addressof(xs), a["tokens"], a["heads"], a["dim"], a["w"], a["w_dt"],
                           a["eps"], a["pos"], a["rates"], a["rot"], a["inter"], a["mag"], a["out"],
                           ctypes.addressof(os_), None) == _mtpk.EINVAL


CACHE = dict(q=P, qs=(2048, 64, 512), k=P, ks=(512, 64, 128), v=P, vs=(512, 64, 128), qn=None, kn=None, ndt=1, eps=1e-6,
             rates=P, rot=64, kp=P, vp=P, rows=160, table=P, stride=10, base=P, keep=None, kb=0, ks_=0, batch=2, t=4, heads=8,
             kvh=2, hd=64, out=P, os=(2048, 64, 512))


@pytest.mark.parametrize("bad", [
    {"q": None}, {"k": None}, {"v": P + 8}, {"kp": None}, {"vp": P + 2}, {"rows": 0}, {"rows": 161}, {"table": None},
    {"stride": 0}, {"base": None}, {"keep": P, "kb": -1}, {"batch": -1}, {"t": 0}, {"heads": 0}, {"kvh": 0}, {"hd": 4},
    {"rot": 65}, {"qs": (2048, 60, 512)}, {"vs": (508, 64, 128)}, {"os": (2048, 64, 511)}, {"qn": P, "ndt": 4},
    {"batch": 1 << 20, "t": 1 << 20},
])  # fmt: skip
def test_rotate_to_cache_refuses(lib, bad) -> None:
    a = {**CACHE, **bad}
    st = [_arr(*a[n]) for n in ("qs", "ks", "vs", "os")]
    qs, ks, vs, os_ = (ctypes.addressof(s) for s in st)
    assert lib.mtpk_rotate_to_cache(
        a["q"], qs, a["k"], ks, a["v"], vs, a["qn"], a["kn"], a["ndt"], a["eps"], a["rates"], a["rot"], 0, 1.0, a["kp"], a["vp"],
        a["rows"], a["table"], a["stride"], a["base"], None, a["keep"], a["kb"], a["ks_"], a["batch"], a["t"], a["heads"],
        a["kvh"], a["hd"], a["out"], os_, None) == _mtpk.EINVAL
