"""Plain 64-bit forms of the grouped products, and the bounds their tests use."""
from __future__ import annotations

import numpy as np

# Half a step of a rounding to the type, relative to the value; and the spacing
# of its subnormals, halved.
HALF_STEP = {"bfloat16": 2.0 ** -8, "float16": 2.0 ** -11, "float32": 2.0 ** -24}
TINY = {"bfloat16": 2.0 ** -134, "float16": 2.0 ** -25, "float32": 2.0 ** -150}


def clean_offsets(offsets, rows):
    """What the kernels make of offsets: clamped to the rows and to the largest before."""
    return np.maximum.accumulate(np.clip(np.asarray(offsets, np.int64), 0, rows))


def rows_form(A, B, trans, offsets, alpha, beta, C):
    """(C, sum of |terms|) of the rows form in float64; A m x k, B groups x ..., C m x n."""
    out, mag = C.copy(), np.zeros_like(C)
    off = clean_offsets(offsets, A.shape[0])
    for g in range(len(off) - 1):
        r = slice(off[g], off[g + 1])
        op = B[g].T if trans else B[g]
        acc = alpha * (A[r] @ op) if alpha else np.zeros_like(C[r])
        out[r] = acc + (beta * C[r] if beta else 0.0)
        mag[r] = abs(alpha) * (np.abs(A[r]) @ np.abs(op))
    return out, mag


def inner_form(A, B, offsets, alpha, beta, C):
    """The same of the inner form; A k x m, B k x n, C groups x m x n."""
    out, mag = C.copy(), np.zeros_like(C)
    off = clean_offsets(offsets, A.shape[0])
    for g in range(len(off) - 1):
        r = slice(off[g], off[g + 1])
        acc = alpha * (A[r].T @ B[r]) if alpha else np.zeros_like(C[g])
        out[g] = acc + (beta * C[g] if beta else 0.0)
        mag[g] = abs(alpha) * (np.abs(A[r]).T @ np.abs(B[r]))
    return out, mag


def bound(want, mag, k, beta, C, ctype):
    """How far a right result may be. Products of two 16-bit floats are exact in
    32 bits; each of the at most k additions is off by at most one step (a
    truncation: 2^-23) of a partial sum no larger than `mag`; scaling by alpha
    and adding beta * C round once more each; the result is rounded once to
    its type."""
    acc = (k + 3) * 2.0 ** -23 * (mag + np.abs(beta * C))
    return acc + HALF_STEP[ctype] * (np.abs(want) + acc) + TINY[ctype]


def assert_close(got, want, mag, k, beta, C, ctype, where=None):
    err = np.abs(got - want)
    lim = bound(want, mag, k, beta, C, ctype)
    ok = (err <= lim) | (np.isnan(got) & np.isnan(want))
    if not ok.all():
        i = np.unravel_index(np.argmin(ok), ok.shape)
        raise AssertionError(f"{where}: {np.count_nonzero(~ok)} of {ok.size} outside; first at {i}: got {got[i]}, "
                             f"want {want[i]}, off {err[i]:.3g}, bound {lim[i]:.3g}")
