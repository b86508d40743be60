"""Attention over the paged cache where the factor of the scores leaves the range of ordinary numbers: scales and f32 query
rows whose product with each other is ordinary, or zero, while one of them is not.  Against the formula in 64 bits with the
bounds of tests/paged_util.py."""
import numpy as np
import pytest

from tests.paged_util import attention64, make_case

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def be():
    import allpaka_amd as apk

    b = apk.Backend(0)
    yield b
    b.close()


def check(be, c, scale, window=0):
    """both entries, where every sequence brings one row; else the chunks'"""
    scale = float(np.float32(scale))  # as the entries take it
    want, tol = attention64(c, scale, window)
    t = {k: torch.from_numpy(np.ascontiguousarray(c[k])).cuda() for k in ("q", "K", "V", "table", "q_off", "kv_len")}
    args, heads = (t["K"], t["V"], c["page"], t["table"]), (c["n_q"], c["n_kv"], c["hd"], scale)
    got = [be.attend_paged_chunk(t["q"], *args, t["q_off"], t["kv_len"], *heads, window=window)]
    if len(c["q"]) == len(c["kv_len"]):
        got.append(be.attend_paged(t["q"], *args, t["kv_len"], *heads, window=window))
    assert be.take_faults() == 0
    for g in got:
        g = g.cpu().numpy().astype(np.float64)
        assert np.all(np.isfinite(g)), f"{np.count_nonzero(~np.isfinite(g))} of {g.size} values are not finite"
        err = np.abs(g - want)
        assert np.all(err <= tol), f"worst {np.max(err / tol):.2f} of the bound"


def case(seed, hd, new, f16=False):
    """lengths that end inside a block of keys, and rows that do not see the last ones"""
    return make_case(seed, [50, 9, 131], new, 4, 2, hd, 16, f16)


# scores that are all (next to) zero: the plain mean of the values
@pytest.mark.parametrize("hd", [64, 128, 256, 48])
@pytest.mark.parametrize("new", [[1, 1, 1], [4, 2, 40]], ids=["tokens", "chunks"])
@pytest.mark.parametrize("scale,size", [(0.0, 1e-12), (0.0, 1e-20), (0.0, 1e-36), (0.0, 1e-42), (0.0, 0.0), (1e-9, 1e-36), (-1e-20, 1e-30), (1e-42, 1e-12)])
def test_scores_that_vanish(be, hd, new, scale, size):
    c = case(700 + hd, hd, new)
    c["q"] *= np.float32(size)
    check(be, c, scale)
    check(be, c, scale, window=20)


# ordinary scores out of factors that are not
@pytest.mark.parametrize("hd", [64, 128, 256, 48])
@pytest.mark.parametrize("new", [[1, 1, 1], [4, 2, 40]], ids=["tokens", "chunks"])
@pytest.mark.parametrize("scale,size", [(1e-33, 1e32), (1e-38, 1e37), (-1e-40, 1e37), (1e37, 1e-38), (3e38, 1e-39)])
def test_scores_of_factors_far_apart(be, hd, new, scale, size):
    c = case(710 + hd, hd, new)
    c["q"] = (c["q"] * np.float64(size)).astype(np.float32)
    check(be, c, scale)


def test_tiny_scales_of_fp16_rows(be):
    for hd in (64, 128, 256, 48):
        for new in ([1, 1, 1], [4, 2, 40]):
            for scale in (0.0, 1e-38, -1e-44):
                check(be, case(720 + hd, hd, new, True), scale)
