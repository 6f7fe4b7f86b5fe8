"""The 8-bit row forms and the attention over rows in 64 bits, in numpy, for the tests.

Written from the definitions in include/kvx/kvx_attn.h, apart from the kernels."""
import numpy as np

LATENT, ROPE, DIM, GROUP = 512, 64, 576, 32
CODES = {"none": 0, "latent": 512, "row": 576}
ROW_BYTES = {"none": 1152, "latent": 768, "row": 640}


def _code_values():
    v = np.empty(128)
    for b in range(128):
        e, f = b >> 3, b & 7
        v[b] = (8 + f) * 2.0 ** (e - 10) if e else f * 2.0 ** -9
    v[127] = np.nan
    return v


CODE_VALUES = np.concatenate([_code_values(), -_code_values()])


def e4m3(x):
    """Codes of float64 values: nearest, ties to the even code; NaN 127 (sign kept)."""
    mag = np.minimum(np.abs(x), 448.0)
    grid = CODE_VALUES[:127]
    hi = np.clip(np.searchsorted(grid, mag), 1, 126)
    lo = hi - 1
    below, above = mag - grid[lo], grid[hi] - mag
    pick = np.where((above < below) | ((above == below) & (hi % 2 == 0)), hi, lo)
    pick = np.where(np.isnan(x), 127, pick)
    return (pick + 128 * np.signbit(x)).astype(np.uint8)


def encode(bits, values, quant):
    """uint8 [n, row bytes] of rows given as their 16-bit patterns (uint16 [n, 576]) and float64 values."""
    n = values.shape[0]
    if quant == "none":
        return np.ascontiguousarray(bits).view(np.uint8).reshape(n, -1)
    d = CODES[quant]
    rec = np.zeros((n, ROW_BYTES[quant]), np.uint8)
    g = values[:, :d].reshape(n, d // GROUP, GROUP)
    top = np.where(np.isfinite(g), np.abs(g), 0.0).max(axis=2)
    e = np.full(top.shape, -127)
    for i in np.ndindex(top.shape):
        if top[i] > 0:
            while top[i] > 448.0 * 2.0 ** e[i]:
                e[i] += 1
    with np.errstate(invalid="ignore"):
        rec[:, :d] = e4m3(g / 2.0 ** e[:, :, None]).reshape(n, d)
    end = d + 2 * (DIM - d)
    rec[:, d:end] = np.ascontiguousarray(bits[:, d:]).view(np.uint8).reshape(n, -1)
    rec[:, end:end + d // GROUP] = e + 127
    return rec


def decode(rec, raw_values, quant):
    """float64 [n, 576] of rows; raw_values: of the 16-bit patterns (uint16 array -> float64 array)."""
    rec = np.ascontiguousarray(rec)
    if quant == "none":
        return raw_values(rec.view(np.uint16))
    d = CODES[quant]
    end = d + 2 * (DIM - d)
    g = CODE_VALUES[rec[:, :d]].reshape(-1, d // GROUP, GROUP)
    x = (g * 2.0 ** (rec[:, end:end + d // GROUP].astype(np.float64) - 127)[:, :, None]).reshape(-1, d)
    return np.concatenate([x, raw_values(np.ascontiguousarray(rec[:, d:end]).view(np.uint16))], axis=1)


def keys_of(slots, draft_slots, tree_mask, stride, hot_rows):
    """Per request: hot rows of the keys that exist, and which of the tokens sees each (bool [tokens, keys])."""
    for b in range(slots.shape[0]):
        rows, seen = [], []
        tokens = 1 if draft_slots is None else draft_slots.shape[1]
        for s in slots[b]:
            if s >= 0 and b * stride + int(s) < hot_rows:
                rows.append(b * stride + int(s))
                seen.append([True] * tokens)
        if draft_slots is not None:
            for j, s in enumerate(draft_slots[b]):
                if s >= 0 and b * stride + int(s) < hot_rows:
                    rows.append(b * stride + int(s))
                    mask = tree_mask[b] if tree_mask is not None else [(2 << t) - 1 for t in range(tokens)]
                    seen.append([bool((int(m) >> j) & 1) for m in mask])
        yield np.array(rows, np.int64), np.array(seen, bool).reshape(len(rows), tokens).T


def attention(q, rows_of, keys, scale):
    """float64 (out, lse, weighted, score error) for q [reqs, tokens, heads, 576].

    rows_of(hot rows) gives float64 rows.  ``weighted`` is sum p |v| and the last, per query, sum over the 576 products
    of |q k| at its largest key: what the error bounds are made of."""
    B, T, H, _ = q.shape
    out, lse = np.zeros((B, T, H, LATENT)), np.full((B, T, H), -np.inf)
    weighted, size = np.zeros((B, T, H, LATENT)), np.zeros((B, T, H))
    for b, (rows, seen) in enumerate(keys):
        k = rows_of(rows)
        for t in range(T):
            use = k[seen[min(t, seen.shape[0] - 1)]] if len(rows) else k[:0]
            if not len(use):
                continue
            s = q[b, t] @ use.T * scale
            top = s.max(axis=1, keepdims=True)
            p = np.exp(s - top)
            total = p.sum(axis=1, keepdims=True)
            lse[b, t] = (top + np.log(total))[:, 0]
            p /= total
            out[b, t], weighted[b, t] = p @ use[:, :LATENT], p @ np.abs(use[:, :LATENT])
            size[b, t] = (np.abs(q[b, t]) @ np.abs(use.T) * abs(scale)).max(axis=1)
    return out, lse, weighted, size
