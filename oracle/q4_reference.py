"""The 4-bit layout, the products and the norm in numpy and 64 bits, from their definitions (no GPU, no library)."""
import numpy as np

NIBBLE = [0, 4, 1, 5, 2, 6, 3, 7]              # of a word, for columns 0..7 of it


def tiles(N, K):
    return -(-N // 16), -(-K // 128)


def pack(code, scale, zero, group, pad_code=8, pad_scale=0.0, pad_zero=8):
    """code N x K, scale and zero N x ceil(K / group) -> (codes, scales, zeros) as the device holds them, flat."""
    N, K = code.shape
    nt, kt = tiles(N, K)
    q = np.full((nt * 16, kt * 128), pad_code, np.uint32)
    q[:N, :K] = code
    q = q.reshape(nt, 16, kt, 4, 4, 8)          # [row tile][row][column tile][j][kg][column]
    words = np.zeros((nt, 16, kt, 4, 4), np.uint32)
    for o in range(8):
        words |= q[..., o] << np.uint32(4 * NIBBLE[o])
    codes = np.ascontiguousarray(words.transpose(0, 2, 4, 1, 3)).view(np.uint8).reshape(-1)
    per = 128 // group

    def per_group(v, pad, dtype):
        full = np.full((nt * 16, kt * per), pad, dtype)
        full[:N, :v.shape[1]] = v
        return np.ascontiguousarray(full.reshape(nt, 16, kt, per).transpose(0, 2, 1, 3)).reshape(-1)
    return codes, per_group(scale, pad_scale, np.float16), None if zero is None else per_group(zero, pad_zero, np.uint8)


def unpack(codes, scales, zeros, N, K, group):
    """The inverse, element by element from the header's words: (code, scale, zero) as above."""
    nt, kt = tiles(N, K)
    per = 128 // group
    n, k = np.arange(N)[:, None], np.arange(K)[None, :]
    word = codes.view(np.uint32)[(((n // 16 * kt + k // 128) * 4 + k % 32 // 8) * 16 + n % 16) * 4 + k % 128 // 32]
    code = (word >> np.uint32(4) * np.array(NIBBLE, np.uint32)[k % 8]) & np.uint32(15)
    g = np.arange(-(-K // group))[None, :]
    at = ((n // 16 * kt + g // per) * 16 + n % 16) * per + g % per
    return code.astype(np.int64), scales[at], None if zeros is None else zeros[at].astype(np.int64)


def values(code, scale, zero, group):
    """What the parts stand for, in 64 bits."""
    K = code.shape[1]
    at = np.arange(K) // group
    z = 8 if zero is None else zero[:, at]
    return (code - z).astype(np.float64) * scale.astype(np.float64)[:, at]


def quantize(W, group, zeros):
    """(code, scale, zero) of W by the definition; the scale in fp32 and then fp16, the rest in 64 bits."""
    N, K = W.shape
    G = -(-K // group)
    code = np.full((N, K), 8, np.int64); scale = np.zeros((N, G), np.float16); zero = np.full((N, G), 8, np.int64)
    for g in range(G):
        w = W[:, g * group:(g + 1) * group].astype(np.float32)
        bad = ~np.isfinite(w).all(1)
        wf = np.where(np.isfinite(w), w, 0).astype(np.float32)
        with np.errstate(over="ignore"):
            if zeros:
                lo, hi = np.minimum(wf.min(1), 0), np.maximum(wf.max(1), 0)
                s = (hi - lo) / np.float32(15)
            else:
                s = np.abs(wf).max(1) / np.float32(7)
            s = np.minimum(s, np.float32(65504)).astype(np.float16)
        some = (s > 0) & ~bad
        d = np.where(some, s, 1).astype(np.float64)
        z = np.where(some, np.clip(np.rint(-lo.astype(np.float64) / d), 0, 15), 8) if zeros else np.full(N, 8.0)
        q = np.clip(np.rint(wf.astype(np.float64) / d[:, None]) + z[:, None], 0, 15)
        code[:, g * group:(g + 1) * group] = np.where(some[:, None], q, z[:, None])
        scale[:, g] = np.where(bad, np.float16(np.nan), s)
        zero[:, g] = z
    return code, scale, zero if zeros else None


def rmsnorm(x, residual, weight, eps, q8):
    """(sum, y or codes, scales): sum in the rows' type, y and scales in 64 bits."""
    t = x.dtype
    h = x if residual is None else (x.astype(np.float64) + residual.astype(np.float64)).astype(t)
    hd, wd = h.astype(np.float64), weight.astype(np.float64)
    with np.errstate(all="ignore"):
        rho = 1 / np.sqrt((hd * hd).mean(1, keepdims=True) + eps)
        p = hd * wd
        if not q8:
            return h, p * rho, None
        top = np.abs(p).max(1)
        top = np.where(np.isfinite(p).all(1), top, np.nan)
        codes = np.where((top > 0)[:, None], np.rint(127 * p / np.where(top > 0, top, 1)[:, None]), 0)
        return h, np.nan_to_num(codes).astype(np.int64), np.where(top == 0, 0.0, top * rho[:, 0] / 127)


def product(x, xs, w, C, alpha, beta, group, f32):
    """(expected in 64 bits, bound of the error) of every output of a product with 4-bit weights of values w.

    The bound: code - zero is a whole number of at most 5 bits, its product with an fp16 is exact in fp32,
    the inner sum of an int8 group is exact altogether.  An output is a sum of K products in fp32 in some order: a group's
    (`group` additions), the groups' (one fma each), and the pieces' of K (up to 64 here), each addition off by at most 2^-23 of
    the sums of magnitudes (half of that where it rounds, all of it where a matrix instruction should cut off), so
    |error| <= (group + groups + 64) 2^-23 sum |x w|.  int8: (groups + 64) 2^-23 and one more rounding by x_scales.  alpha, beta
    and C: two roundings, 2^-23 (|alpha acc| + |beta c|).  The result's own rounding: half a step, 2^-11 |y| and half of the
    smallest fp16, 2^-25."""
    xd = x.astype(np.float64) if xs is None else x.astype(np.float64) * xs.astype(np.float64)[:, None]
    K = x.shape[1]
    groups = -(-K // group) if K else 0
    acc, mag = xd @ w.T, np.abs(xd) @ np.abs(w).T
    adds = groups + 64 + (group if xs is None else 2)
    tol = adds * 2.0 ** -23 * mag
    y = acc
    if C is not None:
        c = np.broadcast_to(C.astype(np.float64), acc.shape)
        y = alpha * acc + beta * c
        tol = abs(alpha) * tol + 2.0 ** -23 * (np.abs(alpha * acc) + abs(alpha) * tol + np.abs(beta * c))
    tol = tol + (2.0 ** -24 * np.abs(y) if f32 else 2.0 ** -11 * (np.abs(y) + tol) + 2.0 ** -25)
    return y, tol
