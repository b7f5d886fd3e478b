"""The top-k of 4-bit matrices on every route of its selection, against 64-bit numpy.

Routes, for s SMs (148 on a B200): at most 2 s rows take 1,024 threads a row; at least 24 s rows of at
most 1,024 keys (24 for every 768 rows of b) and 96 k rows of b take a warp a row; the others 128 threads.
A block's unit of keys is one key up to 2,048 keys (4,096 with 1,024 threads), one vector of 8 up to 8
times as many, several vectors beyond."""
import numpy as np
import pytest

import _fp4_ref as ref
from test_gpu_fp4_limits import _matrix, _random

pytestmark = pytest.mark.gpu


def _best(va, vb, k, skip, fmt):
    """ref.topk of one row, sorting only what reaches the k-th value."""
    p = np.zeros(len(vb))
    for c in range(0, len(va), ref.BLOCK[fmt]):
        p = p + vb[:, c:c + ref.BLOCK[fmt]] @ va[c:c + ref.BLOCK[fmt]]
    p = np.where(np.isnan(p), -np.inf, p)
    if skip is not None:
        p[skip] = -np.inf
    bar = np.partition(p, len(p) - k)[len(p) - k] if k < len(p) else -np.inf
    cols = np.nonzero((p >= bar) & (p > -np.inf))[0]
    o = cols[np.lexsort((cols, -p[cols]))][:k]
    idx, val = np.full(k, -1, np.int32), np.full(k, -np.inf, np.float32)
    idx[:len(o)], val[:len(o)] = o, p[o].astype(np.float32)
    return idx, val


def _check(a, b, va, vb, top, fmt, rows, first=None):
    """va: the values of the queries named in ``rows`` alone."""
    import rfx_b200
    idx, val = rfx_b200.fp4_topk(a, b, top, self_offset=first)
    rfx_b200.fp4_status()
    idx, val = idx.cpu().numpy(), val.cpu().numpy()
    for v, i in zip(va, rows):
        wi, wv = _best(v, vb, top, None if first is None else first + int(i), fmt)
        assert np.array_equal(idx[i], wi) and np.array_equal(val[i], wv), i


def _sample(rng, m, *more):
    return np.unique([0, m - 1, *(i for i in more if i < m), *rng.integers(0, m, 8)])


def _case(fmt, m, n, k, top, kind):
    rng = np.random.default_rng(m + n + k + top)
    c, s = _random(rng, n, k, fmt)
    if kind == "copies":  # some rows equal others
        to, of = rng.integers(0, n, 3000), rng.integers(0, n, 3000)
        c[to], s[to] = c[of], s[of]
    elif kind in ("ties", "equal"):  # five rows, or one, all over
        which = rng.integers(0, 5 if kind == "ties" else 1, n)
        c, s = c[which], s[which]
    elif kind == "extreme":
        s[rng.integers(0, n, n // 50 + 1), 0] = 255 if fmt == "mxfp4" else 127
        s[50:90] = rng.integers(0, 8, (len(s[50:90]), s.shape[1]))
        s[100:110] = rng.integers(180, 200, (len(s[100:110]), s.shape[1])) if fmt == "mxfp4" else 126
    b = _matrix(c, s, k, fmt)
    own = m <= n
    rows = _sample(rng, m, *(range(48, 54) if kind == "extreme" else ()), *(range(99, 103) if kind == "extreme" else ()))
    if own:  # queries: rows of b from a tile's start, themselves left out
        first = (n - m) // 2 // 128 * 128 if kind != "extreme" else 0
        a, ca, sa = b.rows(first, first + m), c[first:first + m], s[first:first + m]
    else:
        first = None
        ca, sa = _random(rng, m, k, fmt)
        a = _matrix(ca, sa, k, fmt)
    with np.errstate(all="ignore"):
        _check(a, b, ref.values(ca[rows], sa[rows], 1.0, fmt), ref.values(c, s, 1.0, fmt), top, fmt, rows, first)


@pytest.mark.parametrize("fmt,n,k,top,kind", [
    ("nvfp4", 6144, 20, 64, "copies"), ("nvfp4", 6200, 64, 64, "equal"), ("mxfp4", 6144, 33, 64, "equal"),
    ("mxfp4", 9000, 200, 64, "ties"), ("nvfp4", 32256, 256, 64, "copies"), ("mxfp4", 32256, 256, 50, "ties"),
    ("nvfp4", 32256, 256, 64, "extreme"), ("mxfp4", 8000, 130, 50, "extreme"), ("nvfp4", 100, 64, 1, "copies"),
    ("mxfp4", 96, 33, 1, "equal")])
def test_a_warp_a_row(fmt, n, k, top, kind):
    _case(fmt, 3700, n, k, top, kind)


@pytest.mark.parametrize("fmt,m,n,k,top,kind", [
    # 128 threads: one key a unit, one vector, several
    ("nvfp4", 300, 65280, 40, 64, "ties"), ("nvfp4", 300, 70000, 64, 33, "ties"), ("mxfp4", 300, 70000, 20, 64, "equal"),
    ("nvfp4", 310, 600000, 16, 50, "copies"), ("mxfp4", 300, 600000, 40, 64, "ties"), ("nvfp4", 300, 600000, 64, 64, "extreme"),
    # the same of 1,024 threads
    ("mxfp4", 5, 131000, 40, 64, "ties"), ("nvfp4", 296, 140000, 20, 64, "ties"), ("mxfp4", 2, 140000, 64, 33, "equal"),
    ("nvfp4", 3, 1100000, 20, 64, "ties"), ("mxfp4", 1, 1100000, 16, 64, "equal")])
def test_a_block_a_row(fmt, m, n, k, top, kind):
    _case(fmt, m, n, k, top, kind)


@pytest.mark.parametrize("m", [4300, 4700, 8600])
def test_several_batches(m):
    """Keys of 1,000,000 rows: 4,224 queries a batch.  The second (and third) reuse the keys' memory,
    begin in the middle of the queries, and here also take another number of threads a row."""
    rng = np.random.default_rng(m)
    n, k, top = 1000000, 16, 20
    c, s = _random(rng, n, k, "nvfp4")
    which = rng.integers(0, n, 400000)
    c[:400000], s[:400000] = c[which], s[which]  # copies
    first = 128 * 3000
    rows = np.unique([0, 4223, 4224, 4225, 4299, min(8447, m - 1), min(8448, m - 1), m - 1])
    b = _matrix(c, s, k, "nvfp4")
    va = ref.values(c[first + rows], s[first + rows], 1.0, "nvfp4")
    _check(b.rows(first, first + m), b, va, ref.values(c, s, 1.0, "nvfp4"), top, "nvfp4", rows, first)


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("m", [8, 130])
@pytest.mark.parametrize("k", [16, 64, 130, 256])
def test_accumulators_within_the_bound(fmt, m, k):
    """What makes the selection exact: an fp32 accumulator of up to 256 columns lies within 2^-15 |a| |b|
    (and 1e-37, for accumulators that vanish) of the product in 64 bits.  Scales over few binades and
    over many, products that cancel, scales whose products are near the smallest normal float."""
    import rfx_b200
    rng = np.random.default_rng(m + k)
    n, worst = 3000, 0.0
    for kind in ("even", "wide", "cancel", "small"):
        spread = {"even": 1, "wide": 30 if fmt == "mxfp4" else 6, "cancel": 3, "small": 4}[kind]
        (ca, sa), (cb, sb) = _random(rng, m, k, fmt, spread), _random(rng, n, k, fmt, spread)
        if kind == "cancel":  # the second half of the columns takes back most of the first
            h = k // 2 // 32 * 32
            if h:
                u = h // ref.BLOCK[fmt]
                ca[:, h:2 * h], sa[:, u:2 * u] = ca[:, :h], sa[:, :u]
                cb[:, h:2 * h], sb[:, u:2 * u] = cb[:, :h] ^ 8, sb[:, :u]
                cb[:, h] ^= 1
        if kind == "small":
            if fmt == "nvfp4":
                sa[:], sb[:] = rng.integers(1, 9, sa.shape), rng.integers(1, 9, sb.shape)
            else:
                sa[:], sb[:] = rng.integers(60, 68, sa.shape), rng.integers(60, 68, sb.shape)  # 2^-67 to 2^-60
        va, vb = ref.values(ca, sa, 1.0, fmt), ref.values(cb, sb, 1.0, fmt)
        got = rfx_b200.fp4_product(_matrix(ca, sa, k, fmt), _matrix(cb, sb, k, fmt)).double().cpu().numpy()
        rfx_b200.fp4_status()
        size = np.linalg.norm(va, axis=1)[:, None] * np.linalg.norm(vb, axis=1)[None]
        off = np.abs(got - va @ vb.T)
        assert (off <= 2.0 ** -15 * size + 1e-37).all(), (kind, (off / size).max())
        if kind != "small":
            worst = max(worst, float((off[size > 0] / size[size > 0]).max()))
    print(f"largest error / (|a| |b|): 2^{np.log2(max(worst, 2.0 ** -60)):.1f}")


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("m,begin,end", [(3, 128, 129), (5, 256, 2011), (400, 128, 1500), (3700, 384, 3999)])
def test_a_view_as_rows(fmt, m, begin, end):
    """The rows searched are a view that starts at a later tile and ends inside one; what lies outside
    (rows of larger norms, rows of NaN) is neither found nor felt."""
    rng = np.random.default_rng(m + begin + end)
    n, k, top = 4000, 72, 12
    c, s = _random(rng, n, k, fmt)
    va_c, va_s = _random(rng, m, k, fmt)
    out = np.r_[0:begin, end:n]
    s[out] += 40 if fmt == "nvfp4" else 20
    s[rng.choice(out, 30), 0] = 127 if fmt == "nvfp4" else 255
    s[min(end, n - 1), 1] = 127 if fmt == "nvfp4" else 255  # in the view's last tile
    b = _matrix(c, s, k, fmt)
    a = _matrix(va_c, va_s, k, fmt)
    rows = _sample(rng, m)
    _check(a, b.rows(begin, end), ref.values(va_c[rows], va_s[rows], 1.0, fmt), ref.values(c[begin:end], s[begin:end], 1.0, fmt),
           top, fmt, rows)
