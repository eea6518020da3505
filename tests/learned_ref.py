"""Plain forms in 64 bits of the learned layers (gated recurrence, grouped products, 8-bit product), with the rounding errors
that a kernel which holds everything in f32 and rounds once may make: each function returns (value, bound) arrays, the bound
being a first-order sum of half steps.  Test infrastructure."""
import numpy as np

U = 2.0 ** -24                                    # half a step of f32, relative
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}   # half a step of the type: eps / 2
TINY = {"f32": 0.0, "f16": 2.0 ** -25, "bf16": 0.0}                          # half of f16's smallest step


def out_bound(v, err, dtype):
    """Bound after the one rounding to the output's type."""
    return err + HALF[dtype] * (np.abs(v) + err) + TINY[dtype]


def gate(g, sigmoid):
    """(a, 1 - a, relative error of both): 1 / (1 + exp(-g)) through exp(-|g|): the argument's rounding moves exp by |g| half
    steps, the exponential, the sum, the reciprocal and the product by at most two half steps each (1 ulp functions)."""
    if not sigmoid:
        return g, np.ones_like(g), np.zeros_like(g)
    e = np.exp(-np.abs(g))
    r = 1 / (1 + e)
    return np.where(g >= 0, r, e * r), np.where(g >= 0, e * r, r), U * (10 + 2 * np.abs(g))


def scan(g, x, off, h0, sigmoid):
    """h, h_last and their bounds; one multiply-add (and the gate's error) per frame, passed on by the gates.  A state that
    crosses a piece is multiplied by the piece's product of gates: one more rounding per gate, the same sum once more."""
    n, D = len(off) - 1, x.shape[1]
    a, na, ra = gate(g, sigmoid)
    h, eh = np.zeros_like(x), np.zeros_like(x)
    prev, eprev = np.zeros_like(x), np.zeros_like(x)
    last, elast = np.zeros((n, D)), np.zeros((n, D))
    for u in range(n):
        s = np.zeros(D) if h0 is None else h0[u].astype(np.float64)
        e = np.zeros(D)
        for t in range(off[u], off[u + 1]):
            prev[t], eprev[t] = s, e
            b = na[t] * x[t]
            e = np.abs(a[t]) * e + (ra[t] + 3 * U) * (np.abs(a[t] * s) + np.abs(b)) + U * np.abs(a[t] * s + b)
            s = a[t] * s + b
            h[t], eh[t] = s, e
        last[u], elast[u] = s, e
    return dict(h=h, eh=eh, last=last, elast=elast, prev=prev, eprev=eprev, a=a, na=na, ra=ra)


def scan_back(f, g, x, off, dh, dlast, sigmoid):
    n, D = len(off) - 1, x.shape[1]
    a, na, ra = f["a"], f["na"], f["ra"]
    lam, el = np.zeros_like(x), np.zeros_like(x)
    d0, e0 = np.zeros((n, D)), np.zeros((n, D))
    for u in range(n):
        c = np.zeros(D) if dlast is None else dlast[u].astype(np.float64)
        e = np.zeros(D)
        for t in range(off[u + 1] - 1, off[u] - 1, -1):
            v = dh[t] + c
            ev = e + U * np.abs(v) + U * (np.abs(dh[t]) + np.abs(c))
            lam[t], el[t] = v, ev
            c = a[t] * v
            e = np.abs(a[t]) * ev + (ra[t] + 3 * U) * np.abs(c)
        d0[u], e0[u] = c, e
    if not sigmoid:
        dg = lam * f["prev"]
        return dict(dx=lam, edx=el, dg=dg, edg=el * np.abs(f["prev"]) + np.abs(lam) * f["eprev"] + 3 * U * np.abs(dg), d0=d0, e0=e0)
    diff = f["prev"] - x
    ediff = f["eprev"] + U * (np.abs(f["prev"]) + np.abs(x))
    dx, w = lam * na, a * na
    dg = lam * w * diff
    return dict(dx=dx, edx=el * na + np.abs(dx) * (ra + 3 * U), dg=dg,
                edg=el * w * np.abs(diff) + np.abs(lam) * w * ediff + np.abs(dg) * (2 * ra + 6 * U), d0=d0, e0=e0)


def product(p, q, dtype):
    """p @ q in 64 bits (p, q hold exact values of the operands' type) and the bound of an f32 accumulation in any order:
    every product is exact (16-bit types) or half a step off (f32), every one of the k - 1 additions half a step of a partial
    sum that is at most sum |p| |q|."""
    mag = np.abs(p) @ np.abs(q)
    k = p.shape[1]
    return p @ q, U * (k + 1) * mag


def group(x, w, off, bias, dtype):
    y, e = np.zeros((x.shape[0], w.shape[1])), np.zeros((x.shape[0], w.shape[1]))
    for g in range(len(off) - 1):
        r = slice(off[g], off[g + 1])
        v, b = product(x[r], w[g].T, dtype)
        y[r], e[r] = (v, b) if bias is None else (v + bias[g], b + U * np.abs(v + bias[g]))
    return y, e


def group_dw(dy, x, off, dtype):
    n = len(off) - 1
    dw, e = np.zeros((n, dy.shape[1], x.shape[1])), np.zeros((n, dy.shape[1], x.shape[1]))
    db, eb = np.zeros((n, dy.shape[1])), np.zeros((n, dy.shape[1]))
    for g in range(n):
        r = slice(off[g], off[g + 1])
        dw[g], e[g] = product(dy[r].T, x[r], dtype)
        db[g], eb[g] = dy[r].sum(0), U * (off[g + 1] - off[g]) * np.abs(dy[r]).sum(0)
    return dw, e, db, eb


def quantize(x):
    """Scale and codes by definition: f32 maximum / 127, f32 quotient, nearest whole number, ties to even."""
    x = np.asarray(x, np.float32)
    s = np.abs(x).max(1) / np.float32(127)
    with np.errstate(divide="ignore", invalid="ignore"):
        q = np.rint((x / s[:, None]).astype(np.float32))
    return s, np.where(np.isfinite(s[:, None]) & (s[:, None] > 0), q, 0).astype(np.int8)


def i8(xq, xs, wq, ws, bias):
    """The sum is exact; its rounding to f32, two scales, the bias: four half steps."""
    v = (xq.astype(np.int64) @ wq.astype(np.int64).T) * xs[:, None].astype(np.float64) * ws.astype(np.float64)
    y = v if bias is None else v + bias.astype(np.float64)
    return y, 3.01 * U * np.abs(v) + U * np.abs(y)
