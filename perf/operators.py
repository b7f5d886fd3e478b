"""Cases of the microscaled 4-bit operators: quantisation, product and top-k neighbours.

A matrix in 4 bits holds e2m1 codes (sign, then 0, .5, 1, 1.5, 2, 3, 4, 6) with one scale per
block of consecutive columns: "mxfp4" has blocks of 32 with a power of two (e8m0), "nvfp4"
blocks of 16 with an e4m3 scale and one power of two for the whole matrix.

``run`` computes a case in plain torch operations, or, with ``own`` set, through rfx_b200.
"""
import math
import os
import sys

import torch

own = False

BLOCK = {"mxfp4": 32, "nvfp4": 16}
DTYPE = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
MAGS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _rfx():
    path = os.path.abspath("rfx-fuse_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import rfx_b200
    return rfx_b200


def listed():
    return [
        # one new row's factors, quantised before it is compared with the stored ones
        dict(name="quantize-one-row", op="quantize", fmt="nvfp4", rows=1, cols=64, dtype="f32",
             out="f32", pad=0),
        # the rank-64 factors of a million rows
        dict(name="quantize-factors", op="quantize", fmt="nvfp4", rows=1000000, cols=64, dtype="f32",
             out="f32", pad=0),
        # 200,000 rows of 50 columns inside a wider buffer, blocks that end ragged
        dict(name="quantize-ragged", op="quantize", fmt="mxfp4", rows=200000, cols=50, dtype="bf16",
             out="bf16", pad=6),
        # a large dense matrix of odd size
        dict(name="quantize-dense", op="quantize", fmt="mxfp4", rows=8191, cols=4095, dtype="f16",
             out="f32", pad=1),
        # one row of the approximate proximity of a million rows
        dict(name="product-one-row", op="product", fmt="nvfp4", m=1, n=1000000, k=64, out="f32"),
        # a block of proximity rows of 200,000 training rows
        dict(name="product-rows", op="product", fmt="nvfp4", m=1024, n=200000, k=64, out="f32"),
        # odd sizes, the second format, half precision out
        dict(name="product-odd", op="product", fmt="mxfp4", m=777, n=10001, k=200, out="f16"),
        # a few rows against a wide matrix: a long inner axis with few output tiles
        dict(name="product-few-rows", op="product", fmt="nvfp4", m=16, n=8192, k=8192, out="bf16"),
        # a square product that arithmetic bounds
        dict(name="product-square", op="product", fmt="mxfp4", m=8192, n=8192, k=8192, out="bf16"),
        # the neighbours of one new row among a million
        dict(name="topk-one-row", op="topk", fmt="nvfp4", m=1, n=1000000, k=64, top=50, same=False),
        # every row's neighbours among 10,000, itself left out
        dict(name="topk-all-rows", op="topk", fmt="mxfp4", m=10000, n=10000, k=48, top=10, same=True),
        # a slice of the million rows' top-50
        dict(name="topk-slice", op="topk", fmt="nvfp4", m=4096, n=1000000, k=64, top=50, same=True),
    ]


def _log(rng, lo, hi):
    """A whole number spread over [lo, hi] by its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    fmt = rng.choice(["mxfp4", "nvfp4"])
    op = rng.choice(["quantize", "product", "topk"])
    if op == "quantize":
        cols = _log(rng, 1, 4096)
        rows = _log(rng, 1, min(1000000, 64000000 // cols))
        return dict(op=op, fmt=fmt, rows=rows, cols=cols, dtype=rng.choice(["f32", "bf16", "f16"]),
                    out=rng.choice(["f32", "bf16"]), pad=rng.choice([0, 0, 1, 3, 8]))
    if op == "product":
        k = _log(rng, 16, 8192)
        m = _log(rng, 1, 8192)
        n = _log(rng, 16, min(1000000, 67000000 // k, 200000000 // m))
        return dict(op=op, fmt=fmt, m=m, n=n, k=k, out=rng.choice(["f32", "bf16", "f16"]))
    k = _log(rng, 8, 256)
    n = _log(rng, 64, min(1000000, 64000000 // k))
    m = _log(rng, 1, min(10000, 4000000000 // n, 260000000000 // (n * k)))
    return dict(op=op, fmt=fmt, m=m, n=n, k=k, top=rng.randint(1, 64), same=m <= n and rng.random() < 0.5)


# ---- inputs ----------------------------------------------------------------------------

def _factors(rows, cols, gen):
    """Rows like low-rank factors: ten groups around their means, columns of falling weight,
    a few rows that equal others."""
    dev = gen.device
    mean = torch.randn(10, cols, generator=gen, device=dev)
    which = torch.randint(0, 10, (rows,), generator=gen, device=dev)
    x = torch.randn(rows, cols, generator=gen, device=dev).mul_(0.7).add_(mean[which])
    x *= torch.arange(1, cols + 1, device=dev, dtype=torch.float32).pow_(-0.5)
    x /= x.norm(dim=1).mean()
    twins = rows // 100
    if twins:
        of = torch.randint(0, rows, (twins,), generator=gen, device=dev)
        x[torch.arange(twins, device=dev) * 100 + 37] = x[of]
    return x


def _pack(codes):
    """[rows, cols] codes -> two to a byte, the even column in the low half."""
    if codes.shape[1] % 2:
        codes = torch.nn.functional.pad(codes, (0, 1))
    return (codes[:, 0::2] | (codes[:, 1::2] << 4)).contiguous()


def _held(rows, cols, fmt, gen, what):
    """A matrix in 4 bits as a program keeps it: (packed codes, scale bytes, matrix scale)."""
    x = _factors(rows, cols, gen) if what == "factors" else torch.randn(
        rows, cols, generator=gen, device=gen.device)
    codes, scales, g = _quantize(x, fmt)
    return _pack(codes), scales, g


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = dict(case)
    if case["op"] == "quantize":
        buf = torch.zeros(case["rows"], case["cols"] + case["pad"], device="cuda", dtype=DTYPE[case["dtype"]])
        buf[:, :case["cols"]] = _factors(case["rows"], case["cols"], gen)
        s["x"] = buf[:, :case["cols"]]
        return s
    what = "factors" if case["k"] <= 256 else "dense"
    s["b"] = _held(case["n"], case["k"], case["fmt"], gen, what)
    if case["op"] == "topk" and case["same"]:
        # a slice of the same rows, from the middle
        s["first"] = (case["n"] - case["m"]) // 2
        p, sc, g = s["b"]
        s["a"] = (p[s["first"]:s["first"] + case["m"]], sc[s["first"]:s["first"] + case["m"]], g)
    else:
        s["first"] = None
        s["a"] = _held(case["m"], case["k"], case["fmt"], gen, what)
    if own:
        r = _rfx()
        for side in ("a", "b"):
            p, sc, g = s[side]
            s[side] = r.Fp4Matrix.from_parts(p, sc, g, cols=case["k"], format=case["fmt"])
    return s


# ---- one pass --------------------------------------------------------------------------

def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    r = _rfx()
    if s["op"] == "quantize":
        return r.fp4_quantize(s["x"], format=s["fmt"]).dequantize(DTYPE[s["out"]])
    if s["op"] == "product":
        return r.fp4_product(s["a"], s["b"], dtype=DTYPE[s["out"]])
    return r.fp4_topk(s["a"], s["b"], s["top"], self_offset=s["first"])


def _run_plain(s):
    if s["op"] == "quantize":
        codes, scales, g = _quantize(s["x"].float(), s["fmt"])
        return _values(codes, scales, g, s["fmt"]).to(DTYPE[s["out"]])
    a, b = (_values(_unpack(p, s["k"]), sc, g, s["fmt"]) for p, sc, g in (s["a"], s["b"]))
    if s["op"] == "product":
        return torch.matmul(a, b.T).to(DTYPE[s["out"]])
    return _topk(a.double(), b.double(), s["top"], s["first"])


def _power(e):
    """2^e in 64 bits, exactly."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _quantize(x, fmt):
    """(codes uint8 [rows, cols], scale bytes uint8 [rows, blocks], matrix scale) of x.

    mxfp4: the block's scale is the smallest power of two of which its largest magnitude is at
    most 6 times.  nvfp4: the matrix scale g is the smallest power of two of which the largest
    magnitude is at most 6 * 448 times; the block's scale is its largest magnitude / (6 g),
    rounded to e4m3.  Values / scale round to the nearest e2m1, ties to the even code, at most 6.
    """
    rows, cols = x.shape
    bs = BLOCK[fmt]
    nb = (cols + bs - 1) // bs
    if cols % bs:
        x = torch.nn.functional.pad(x, (0, nb * bs - cols))
    x = x.reshape(rows, nb, bs).double()  # quotients next to a border between two codes
    amax = x.abs().amax(2)
    if fmt == "mxfp4":
        m, e = torch.frexp(amax)  # amax = m 2^e, .5 <= m < 1
        e = (e - 2 - (m <= 0.75).int()).clamp(min=-127)
        e = torch.where(amax > 0, e, torch.full_like(e, -127))
        scales = (e + 127).to(torch.uint8)
        v = x * _power(-e)[:, :, None]
        g = 1.0
    else:
        m, e = torch.frexp(amax.amax())
        e = (e - 11 - (m <= 0.65625).int()).clamp(min=-126)
        g = _power(torch.where(amax.amax() > 0, e, torch.zeros_like(e)))
        s8 = (amax / (6.0 * g)).float().to(torch.float8_e4m3fn)
        scales = s8.view(torch.uint8)
        t = s8.double() * g
        v = torch.where(t[:, :, None] > 0, x / torch.where(t > 0, t, torch.ones_like(t))[:, :, None], 0.0)
        g = g.float()
    a = v.abs()
    idx = ((a > 0.25).to(torch.uint8) + (a >= 0.75).to(torch.uint8) + (a > 1.25).to(torch.uint8)
           + (a >= 1.75).to(torch.uint8) + (a > 2.5).to(torch.uint8) + (a >= 3.5).to(torch.uint8)
           + (a > 5.0).to(torch.uint8))
    codes = idx | ((v < 0).to(torch.uint8) << 3)
    return codes.reshape(rows, nb * bs)[:, :cols], scales, g


def _unpack(packed, cols):
    return torch.stack((packed & 15, packed >> 4), dim=2).reshape(packed.shape[0], -1)[:, :cols]


def _values(codes, scales, g, fmt):
    """The fp32 values that codes and scales stand for."""
    table = torch.tensor(MAGS + tuple(-v for v in MAGS), device=codes.device)
    s = (_power(scales.int() - 127).float() if fmt == "mxfp4"
         else scales.view(torch.float8_e4m3fn).float())
    v = table[codes.int()] * s.repeat_interleave(BLOCK[fmt], dim=1)[:, :codes.shape[1]]
    return v * g


def _topk(a, b, k, first):
    """The k largest a_i . b_j of every row i, equal ones by ascending j; with ``first``, row i is
    row first + i of b and left out.  Slots without a neighbour hold -1 and -inf."""
    m, n = a.shape[0], b.shape[0]
    kk = min(k, n)
    step = max(1, (1 << 27) // n)
    col = torch.arange(n, device=a.device, dtype=torch.int32)
    idx = torch.full((m, k), -1, device=a.device, dtype=torch.int32)
    val = torch.full((m, k), -math.inf, device=a.device)
    for r0 in range(0, m, step):
        r1 = min(m, r0 + step)
        v = torch.matmul(a[r0:r1], b.T)
        if first is not None:
            rr = torch.arange(r0, r1, device=a.device)
            v[rr - r0, rr + first] = -math.inf
        kth = v.topk(kk, dim=1).values[:, -1:]
        above = v > kth
        tie = v == kth
        need = kk - above.sum(1, keepdim=True)
        take = above | (tie & (tie.cumsum(1, dtype=torch.int32) <= need))
        j = n - torch.where(take, n - col, torch.zeros_like(col)).topk(kk, dim=1).values
        best, order = v.gather(1, j.long()).sort(dim=1, descending=True, stable=True)
        j = j.gather(1, order)
        idx[r0:r1, :kk] = torch.where(best > -math.inf, j, torch.full_like(j, -1))
        val[r0:r1, :kk] = best.float()
    return idx, val


# ---- what a pass cannot do without ---------------------------------------------------------

def work(case):
    bs = BLOCK[case["fmt"]]

    def held(rows, cols):
        return rows * ((cols + 1) // 2 + (cols + bs - 1) // bs)

    size = {"f32": 4, "bf16": 2, "f16": 2}
    if case["op"] == "quantize":
        n = case["rows"] * case["cols"]
        # x read, the 4-bit matrix written and read, its values written
        return {"bytes": n * (size[case["dtype"]] + size[case["out"]]) + 2 * held(case["rows"], case["cols"]),
                "flops": 4 * n}
    flops = 2 * case["m"] * case["n"] * case["k"]
    held_b = held(case["n"], case["k"])
    held_a = 0 if case.get("same") else held(case["m"], case["k"])
    out = case["m"] * (case["top"] * 8 if case["op"] == "topk" else case["n"] * size[case["out"]])
    return {"bytes": held_a + held_b + out, "flops": flops}


# ---- 64-bit values, from the definition ---------------------------------------------------

def _two_64(e):
    """2^e from a table (the device's pow is off by a rounding, which moves ties)."""
    table = torch.tensor([2.0 ** i for i in range(-160, 161)], device=e.device, dtype=torch.float64)
    return table[e.long() + 160]


def _e2m1_64(codes):
    c = codes.long()
    exp, man = (c >> 1) & 3, (c & 1).double()
    mag = torch.where(exp == 0, man * 0.5, (1 + man * 0.5) * _two_64(exp - 1))
    return torch.where(c >= 8, -mag, mag)


def _scale_64(byte, fmt):
    b = byte.long()
    if fmt == "mxfp4":
        return _two_64(b - 127)
    exp, man = b >> 3, (b & 7).double()
    return torch.where(exp == 0, man * 2.0 ** -9, (8 + man) * _two_64(exp - 10))


def _held_64(parts, cols, fmt):
    packed, scales, g = parts
    codes = torch.empty(packed.shape[0], packed.shape[1] * 2, device=packed.device, dtype=torch.uint8)
    codes[:, 0::2] = packed % 16
    codes[:, 1::2] = packed // 16
    block = torch.arange(cols, device=packed.device) // BLOCK[fmt]
    return _e2m1_64(codes[:, :cols]) * _scale_64(scales, fmt)[:, block] * float(g)


def _near_64(v, grid):
    """The nearest member of ``grid`` (ascending, even places win ties) to each v >= 0."""
    mid = (grid[1:] + grid[:-1]) / 2
    lo = torch.bucketize(v, mid)               # ties below
    hi = torch.bucketize(v, mid, right=True)   # ties above
    return grid[torch.where(lo % 2 == 0, lo, hi)]


def _quantize_64(x, fmt):
    cols = x.shape[1]
    grid = _e2m1_64(torch.arange(8, device=x.device))
    block = torch.arange(cols, device=x.device) // BLOCK[fmt]
    amax = torch.stack([part.abs().amax(1) for part in x.split(BLOCK[fmt], dim=1)], dim=1)
    if fmt == "mxfp4":
        scale = _two_64(torch.ceil(torch.log2(amax / 6)).clamp(min=-127))
        scale = torch.where(amax > 6 * scale, scale * 2, torch.where(amax <= 3 * scale, scale / 2, scale))
        scale = scale.clamp(min=2.0 ** -127)
    else:
        top = float(amax.max())
        g = 1.0
        if top > 0:
            while top > 2688 * g:
                g *= 2
            while top <= 1344 * g and g > 2.0 ** -126:
                g /= 2
        scale = g * _near_64(amax / (6 * g), _scale_64(torch.arange(127, device=x.device), fmt))
    t = scale[:, block]
    q = _near_64(torch.where(t > 0, x.abs() / torch.where(t > 0, t, 1.0), 0.0), grid)
    return torch.sign(x) * q * t


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if case["op"] == "quantize":
        out = torch.empty(case["rows"], case["cols"], device="cuda", dtype=torch.float64)
        if case["fmt"] == "nvfp4":  # the matrix scale needs every row
            out.copy_(_quantize_64(s["x"].double(), case["fmt"]))
        else:
            for r0 in range(0, case["rows"], 65536):
                out[r0:r0 + 65536] = _quantize_64(s["x"][r0:r0 + 65536].double(), case["fmt"])
        return out
    a, b = _held_64(s["a"], case["k"], case["fmt"]), _held_64(s["b"], case["k"], case["fmt"])
    if case["op"] == "product":
        return torch.mm(a, b.t())
    m, n, k = case["m"], case["n"], case["top"]
    idx = torch.full((m, k), -1, device=a.device, dtype=torch.int32)
    val = torch.full((m, k), -math.inf, device=a.device, dtype=torch.float64)
    step = max(1, (1 << 27) // n)
    for r0 in range(0, m, step):
        p = torch.mm(a[r0:r0 + step], b.t())
        rows = p.shape[0]
        if s["first"] is not None:
            i = torch.arange(rows, device=p.device)
            p[i, i + r0 + s["first"]] = -math.inf
        left = n - 1 if s["first"] is not None else n
        kk = min(k, left)
        if kk == 0:
            continue
        bar = torch.kthvalue(p, n - kk + 1, dim=1, keepdim=True).values
        where = torch.nonzero(p >= bar)
        v = p[where[:, 0], where[:, 1]]
        # by row, then value descending, then column: nonzero gives ascending columns
        o = torch.argsort(v, descending=True, stable=True)
        o = o[torch.argsort(where[o, 0], stable=True)]
        row = where[o, 0]
        count = torch.bincount(row, minlength=rows)
        place = torch.arange(len(row), device=row.device) - (count.cumsum(0) - count)[row]
        keep = place < kk
        row, place, o = row[keep] + r0, place[keep], o[keep]
        idx[row, place] = where[o, 1].int()
        val[row, place] = v[o]
    return idx, val
