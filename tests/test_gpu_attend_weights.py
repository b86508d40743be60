"""What every key of a long cache counts for: keys of small weight next to one of large weight, and each key on its own,
seen through a channel that only its value has."""
import numpy as np
import pytest

from tests.paged_util import ceil_div, make_case, slots_of

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def be():
    import allpaka_amd as apk

    b = apk.Backend(0)
    yield b
    b.close()


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def attend(be, c, scale, window, chunk, V):
    args = (dev(c["q"]), dev(c["K"]), V, c["page"], dev(c["table"]))
    tail = (dev(c["kv_len"]), c["n_q"], c["n_kv"], c["hd"], scale)
    got = be.attend_paged_chunk(*args, dev(c["q_off"]), *tail, window=window) if chunk else be.attend_paged(*args, *tail, window=window)
    assert be.take_faults() == 0
    return got.cpu().numpy().astype(np.float64)


# One key weighs 1, its value is zero, and n weigh 2^-bits each: the result is what they bring.
#   A score is 0 or g, exactly, g a number of fp16.  Its argument of exp2 is g * log2(e) - the reference: the constant, the
#   product and the sum are rounded, each by 2^-24 of |x| <= 28: a weight is off by 4 * 28 * ln 2 * 2^-24 relative, and by 2^-21 for exp2.
#   In the sum of the values a weight counts as two fp16, 2^-22 of it, or as one, 2^-11 (chunks of fp16 rows).  In chunks fp16's
#   smallest half step, 2^-25, comes to that where weights are far below the largest one of their unit of 64 keys: the
#   large key of the first unit is 2^8 there, so that the 63 others are off by 2^-33 of it at most.
#   Sums of n <= 200 numbers of one sign in f32, in any order: n * 2^-24 relative, for the values and for the weights.
#   The result: half a step of its type.
@pytest.mark.parametrize("hd", [64, 128, 256, 48])
@pytest.mark.parametrize("f16", [True, False], ids=["f16", "f32"])
@pytest.mark.parametrize("rows", [1, 17, 150])
@pytest.mark.parametrize("bits", [4.4, 8.3, 12.6, 15.7, 18.4, 20.2, 22.6, 25.5, 27.3])
def test_small_weights_next_to_a_large_one(be, hd, f16, rows, bits):
    n = 200
    c = make_case(800, [n], [rows], 2, 1, hd, 16, f16)
    at = slots_of(c["table"][0], n, 16)
    g = float(np.float16(bits * np.log(2)))
    c["q"][:] = 0
    c["q"][:, 0::hd] = 1.0
    c["K"][at], c["V"][at] = 0, 1.0
    c["K"][at[7], 0], c["V"][at[7]] = g, 0.0
    others = n - rows + np.arange(rows)[:, None]  # keys that a row sees, but for the large one
    want = np.broadcast_to(others * np.exp(-g) / (1 + others * np.exp(-g)), (rows, 2 * hd))
    short = c["table"]
    wide = np.pad(short, ((0, 0), (0, 80)), constant_values=-1)  # room for more than 1024 keys: another form of the kernel
    for table, chunk in ((short, False), (short, True), (wide, False), (wide, True)):
        if rows > 1 and not chunk:
            continue
        c["table"] = table
        tiles = table is wide and rows > 1 and hd != 48  # the form of chunks
        rel = 4 * 28 * np.log(2) * 2.0 ** -24 + 2.0 ** -21 + (2.0 ** -11 if f16 and tiles else 2.0 ** -22) + 2 * n * 2.0 ** -24 + (2.0 ** -11 if f16 else 2.0 ** -24)
        tol = rel * want + (63 * 2.0 ** -33 if tiles else 0) + (2.0 ** -25 if f16 else 0)
        got = attend(be, c, 1.0, 0, chunk, dev(c["V"]))
        err = np.abs(got - want)
        assert np.all(err <= tol), f"worst {np.max(err / want):.2e} of the result, {np.max(err / tol):.1f} of the bound"


# (lengths, new rows), n_q, n_kv, hd, page, window: caches cut into many parts and into few, tiles that see them in part, one
# launch (short tables), many sequences, windows whose ends fall anywhere
SEEN = [
    ([9001], [1], 8, 2, 128, 64, 0),
    ([5003, 3, 700], [1, 1, 1], 4, 4, 64, 16, 0),
    ([3001], [1], 5, 1, 256, 33, 0),
    ([900, 77], [1, 1], 4, 2, 128, 16, 0),
    ([6000, 4097], [1, 1], 8, 2, 128, 16, 3333),
    ([9001], [9], 4, 2, 128, 64, 0),
    ([4000, 130], [3, 60], 4, 2, 64, 24, 0),
    ([2600, 1000], [5, 33], 4, 1, 256, 16, 0),
    ([5000, 2050], [40, 3], 4, 2, 128, 16, 1500),
    ([3000], [20], 6, 2, 64, 7, 777),
    ([700, 40], [3, 40], 2, 1, 80, 16, 0),
]


@pytest.mark.parametrize("f16", [True, False], ids=["f16", "f32"])
@pytest.mark.parametrize("i", range(len(SEEN)))
def test_every_key_counts_once(be, i, f16):
    """V is zero but for one key a channel, so that the channel holds that key's weight alone: missing it would be 0, counted
    twice it would be doubled; all keys in turn.  The weights are bounded as in tests/paged_util.py, of one key: 2^-11
    where a weight is rounded to fp16, and 2^-11 of the result; n * 2^-24 for the sum of the weights, below 2^-10 here; scores of magnitude
    below 8 of hd products: 8 * (hd + 8) * 2^-24 < 2^-12.  2^-8 covers them, and half of fp16's smallest step beside it."""
    lens, new, n_q, n_kv, hd, page, window = SEEN[i]
    c = make_case(820 + i, lens, new, n_q, n_kv, hd, page, f16, q_gain=0.5, garbage=0.0)
    scale, group, width = hd ** -0.5, n_q // n_kv, n_kv * hd
    q = c["q"].astype(np.float64)
    weights = []  # per row: [n_q, keys]
    for s, n in enumerate(lens):
        k = c["K"][slots_of(c["table"][s], n, page)].astype(np.float64).reshape(n, n_kv, hd)
        for r in range(c["q_off"][s], c["q_off"][s + 1]):
            p = n - (c["q_off"][s + 1] - r)
            x = np.einsum("jgc,gec->gej", k, q[r].reshape(n_kv, group, hd)).reshape(n_q, n) * scale
            x[:, p + 1:] = -np.inf
            if window:
                x[:, :max(0, p - window + 1)] = -np.inf
            assert np.abs(x[np.isfinite(x)]).max() < 8
            w = np.exp(x)
            weights.append(w / w.sum(axis=1, keepdims=True))
    owner = np.repeat(np.arange(len(lens)), new)
    chunks = (False, True) if max(new) == 1 else (True,)
    for first in range(0, max(lens), width):
        V = torch.zeros(c["V"].shape, dtype=torch.float16, device="cuda")
        for s, n in enumerate(lens):
            m = min(n - first, width)
            if m > 0:
                at = slots_of(c["table"][s], n, page)[first:first + m]
                V[torch.from_numpy(at).cuda(), torch.arange(m, device="cuda")] = 1.0
        want = np.zeros((len(q), n_kv, group, hd))
        for r, w in enumerate(weights):
            part = w[:, first:first + width]
            full = np.zeros((n_q, width))
            full[:, :part.shape[1]] = part
            for g in range(n_kv):
                want[r, g] = full[g * group:(g + 1) * group, g * hd:(g + 1) * hd]
        want = want.reshape(len(q), n_q * hd)
        for chunk in chunks:
            err = np.abs(attend(be, c, scale, window, chunk, V) - want)
            bad = err > 2.0 ** -8 * want + (2.0 ** -25 if f16 else 0)
            assert not bad.any(), f"row {np.argwhere(bad)[0][0]} of sequence {owner[np.argwhere(bad)[0][0]]}, keys from {first} on, channel {np.argwhere(bad)[0][1]}: {bad.sum()} off"


# Levels of weights all along a cache, a different one in every stretch: 2^0, 2^-23, 2^-9, 2^-30 .. of the largest, the values of all
# but one level zero at a time, so that the result is what that level brings.  Stretches of whole units of 64 keys: there
# is no larger weight in a unit, so that its weights keep their bits whatever came before.  Bounds as above, |x| <= 40.
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("f16", [True, False], ids=["f16", "f32"])
@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("order", [[0, 23, 9, 30, 4], [30, 9, 0, 23, 12], [26, 17, 8, 0, 14], [0, 38, 0, 38, 19]])
def test_levels_of_weight(be, hd, f16, rows, order):
    span, page = 192, 16
    n = span * len(order) + 40  # the rows' own keys behind them: of the lowest level, value zero
    c = make_case(810, [n], [rows], 4, 2, hd, page, f16)
    c["table"] = np.pad(c["table"], ((0, 0), (0, 80)), constant_values=-1)
    at = slots_of(c["table"][0], n, page)
    g = np.array([np.float16(-b * np.log(2)) for b in order], np.float64)
    c["q"][:] = 0
    c["q"][:, 0::hd] = 1.0
    c["K"][at] = 0
    c["K"][at, 0] = c["K"][at, hd] = np.float16(-40 * np.log(2))
    for i, x in enumerate(g):
        c["K"][at[span * i:span * (i + 1)], 0] = c["K"][at[span * i:span * (i + 1)], hd] = x
    total = span * np.exp(g).sum()  # the keys behind bring below 2^-34 of it
    for level in sorted(set(order)):
        mine = [i for i, b in enumerate(order) if b == level]
        c["V"][at] = 0
        for i in mine:
            c["V"][at[span * i:span * (i + 1)]] = 1.5
        want = 1.5 * span * np.exp(g[mine]).sum() / total
        rel = 4 * 40 * np.log(2) * 2.0 ** -24 + 2.0 ** -21 + (2.0 ** -11 if f16 and rows > 1 else 2.0 ** -22) + 2 * n * 2.0 ** -24 + (2.0 ** -11 if f16 else 2.0 ** -24)
        if rows == 1:  # below 2^-28 of the largest, a single token's weights have 2^-50 of it
            rel += 2.0 ** -50 / 2.0 ** -level
        got = attend(be, c, 1.0, 0, rows > 1, dev(c["V"]))
        err = np.abs(got - want)
        assert np.all(err <= rel * want + (2.0 ** -25 if f16 else 0)), f"level {level}: worst {np.max(err) / want:.2e} of the result, bound {rel:.2e}"


# Two levels in turn, unit after unit: more often than the reference of the weights follows.  A weight of the lower level is then off by
# 2^-33 of the largest at most, the rest as above.
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("f16", [True, False], ids=["f16", "f32"])
@pytest.mark.parametrize("bits", [11.3, 17.5, 22.2])
def test_levels_that_alternate(be, hd, f16, bits):
    rows, units, page = 40, 30, 16
    n = 64 * units + 64
    c = make_case(811, [n], [rows], 4, 2, hd, page, f16)
    at = slots_of(c["table"][0], n, page)
    g = float(np.float16(-bits * np.log(2)))
    c["q"][:] = 0
    c["q"][:, 0::hd] = 1.0
    c["K"][at] = 0
    low = np.arange(n) // 64 % 2 == 1
    c["K"][at[low], 0] = c["K"][at[low], hd] = g
    behind = np.arange(n) >= 64 * units  # the rows' own keys among them: of next to no weight
    c["K"][at[behind], 0] = c["K"][at[behind], hd] = np.float16(-40 * np.log(2))
    low &= ~behind
    c["V"][at], c["V"][at[low]] = 0, 1.5
    many = int(low.sum())
    want = 1.5 * many * np.exp(g) / (many + many * np.exp(g))
    rel = 4 * 40 * np.log(2) * 2.0 ** -24 + 2.0 ** -21 + (2.0 ** -11 if f16 else 2.0 ** -22) + 2 * n * 2.0 ** -24 + (2.0 ** -11 if f16 else 2.0 ** -24)
    err = np.abs(attend(be, c, 1.0, 0, True, dev(c["V"])) - want)
    # (each of them off by 2^-33, times its value, over the sum of the weights)
    assert np.all(err <= rel * want + 1.5 * 2.0 ** -33 + (2.0 ** -25 if f16 else 0)), f"worst {np.max(err) / want:.2e} of the result"


# Scores of widths from the ordinary to next to one-hot, random, so that the reference of the weights moves at any place: in units
# seen in part and whole, at windows' ends and in odd parts; and a key that outweighs all, first, in the middle or last.
@pytest.mark.parametrize("f16", [True, False], ids=["f16", "f32"])
@pytest.mark.parametrize("gain", [4.0, 12.0, 40.0])
@pytest.mark.parametrize("hd,n_q,n_kv,page,window", [(64, 6, 2, 24, 0), (128, 4, 1, 16, 700), (256, 2, 1, 33, 0), (256, 3, 1, 16, 500), (128, 40, 1, 64, 0)])
def test_wide_scores(be, f16, gain, hd, n_q, n_kv, page, window):
    from tests.paged_util import attention64

    seqs = [(1100, 60), (3, 90), (2500, 2)]
    c = make_case(830 + hd + window, [a + b for a, b in seqs], [b for _, b in seqs], n_q, n_kv, hd, page, f16, q_gain=gain)
    for s, j in ((0, 0), (0, 640), (1, 92)):
        at = c["table"][s][j // page] * page + j % page
        c["K"][at, :hd] = 3.0 * np.sign(c["q"][c["q_off"][s], :hd]).astype(np.float16)
    want, tol = attention64(c, hd ** -0.5, window)
    got = attend(be, c, hd ** -0.5, window, True, dev(c["V"]))
    err = np.abs(got - want)
    assert np.all(err <= tol), f"worst {np.max(err / tol):.2f} of the bound"
