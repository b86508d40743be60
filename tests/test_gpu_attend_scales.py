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


def wide(table):
    """The same with room for more than 1024 keys: the forms of the kernels go by the room that there is."""
    return np.pad(table, ((0, 0), (0, 80)), constant_values=-1)


def check(be, c, scale, window=0):
    """both entries, where every sequence brings one row; else the chunks'; with a short table and a wide one"""
    scale = float(np.float32(scale))  # as the entries take it
    want, tol = attention64(c, scale, window)
    t = {k: torch.from_numpy(np.ascontiguousarray(c[k])).cuda() for k in ("q", "K", "V", "table", "q_off", "kv_len")}
    heads, got = (c["n_q"], c["n_kv"], c["hd"], scale), []
    for table in (t["table"], torch.from_numpy(wide(c["table"])).cuda()):
        args = (t["K"], t["V"], c["page"], table)
        got.append(be.attend_paged_chunk(t["q"], *args, t["q_off"], t["kv_len"], *heads, window=window))
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


@pytest.mark.parametrize("hd", [64, 128, 256, 48])
@pytest.mark.parametrize("new", [[1, 1, 1], [4, 2, 40]], ids=["tokens", "chunks"])
def test_infinite_scores_of_fp16_rows(be, hd, new):
    """A score of -inf is a weight of 0; +inf makes its row NaN and no other; scores that are all -inf give zeros."""
    c = case(730 + hd, hd, new, True)
    c["q"][:, 0::hd] = -np.abs(c["q"][:, 0::hd]) - np.float16(0.25)
    want, tol = attention64(c, 0.1)
    free = [p for p in range(c["n_pages"]) if p not in c["table"]]
    d = dict(c, K=c["K"].copy(), V=c["V"].copy(), kv_len=c["kv_len"] + 16)
    # 16 more keys in front of every sequence: a page of its own, whose K is infinite in a channel that every query has
    for s in range(3):
        d["K"][free[s] * 16:free[s] * 16 + 16] = 1.0
        d["K"][free[s] * 16:free[s] * 16 + 16, 0::hd] = np.inf
        d["V"][free[s] * 16:free[s] * 16 + 16] = 3.0
    d["table"] = np.concatenate([np.array(free[:3], np.int32)[:, None], c["table"]], 1)
    t = {k: torch.from_numpy(np.ascontiguousarray(d[k])).cuda() for k in ("q", "K", "V", "table", "q_off", "kv_len")}

    def run():
        heads, out = (4, 2, hd, 0.1), []
        for table in (t["table"], torch.from_numpy(wide(d["table"])).cuda()):
            out.append(be.attend_paged_chunk(t["q"], t["K"], t["V"], 16, table, t["q_off"], t["kv_len"], *heads))
            if max(new) == 1:
                out.append(be.attend_paged(t["q"], t["K"], t["V"], 16, table, t["kv_len"], *heads))
        assert be.take_faults() == 0
        return [o.cpu().numpy().astype(np.float64) for o in out]

    for got in run():
        assert np.all(np.abs(got - want) <= tol)
    t["q"][1, hd] *= -1  # the second head of row 1
    for got in run():
        bad = np.zeros(got.shape, bool)
        bad[1, hd:2 * hd] = True
        assert np.all(np.isnan(got[bad])) and np.all(np.isfinite(got[~bad]))
    t["q"][1, hd] *= -1
    t["kv_len"].fill_(16)  # nothing else to see
    for got in run():
        seen = np.concatenate([np.arange(m) + 16 - m >= 0 for m in new])
        assert np.all(got[seen] == 0) and np.all(got[~seen] == 0)
