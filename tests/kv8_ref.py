"""The 8-bit KV cache restated in numpy, row by row, from its definition:
scales held in f32, codes from quotients in 64 bits, attention in 64 bits."""
import numpy as np


def need_of(x):
    """The scale that rows x [..., head_dim] of one block and head ask for."""
    m = np.max(np.abs(x.astype(np.float64))) if x.size else 0.0
    if not np.isfinite(m):
        return np.float32(np.nan)
    s = np.float32(m) * (np.float32(1.0) / np.float32(127.0))
    return np.float32(0.0) if s < np.float32(2.0 ** -126) else s


def codes_of(x, s):
    if np.isnan(s) or s == 0:
        return np.zeros(x.shape, np.int8)
    return np.clip(np.rint(x.astype(np.float64) / np.float64(s)), -127, 127).astype(np.int8)


class Cache:
    """One sequence, one layer: codes [2][max_ctx][nkv][hd], scales [2][blocks][nkv]."""

    def __init__(self, nkv, hd, max_ctx, block):
        self.block, self.max_ctx = block, max_ctx
        self.codes = np.zeros((2, max_ctx, nkv, hd), np.int8)
        self.scales = np.zeros((2, -(-max_ctx // block), nkv), np.float32)

    def append(self, pos, k, v):
        """Rows k, v [m, nkv, hd] (f32 values) at positions pos, pos + 1, ..."""
        m = min(len(k), self.max_ctx - pos)
        if m <= 0:
            return
        for which, x in enumerate((k[:m], v[:m])):
            for b in range(pos // self.block, (pos + m - 1) // self.block + 1):
                lo, hi = max(pos, b * self.block), min(pos + m, (b + 1) * self.block)
                for h in range(x.shape[1]):
                    rows = x[lo - pos:hi - pos, h]
                    s = need_of(rows)
                    held = self.scales[which, b, h] if lo > b * self.block else np.float32(0)
                    if np.isnan(held):
                        s = held
                    elif held > 0 and not np.isnan(s):
                        times = 0
                        while np.float64(held) * 2.0 ** times < np.float64(s):
                            times += 1
                        s = np.float32(np.float64(held) * 2.0 ** times)
                        if times:
                            old = self.codes[which, b * self.block:lo, h]
                            self.codes[which, b * self.block:lo, h] = np.rint(old.astype(np.float64) / 2.0 ** times)
                    self.scales[which, b, h] = s
                    self.codes[which, lo:hi, h] = codes_of(rows, s)

    def values(self, which, lo, hi):
        """f32 values of positions [lo, hi): each product rounded once."""
        s = self.scales[which][np.arange(lo, hi) // self.block]
        return self.codes[which, lo:hi].astype(np.float32) * s[:, :, None]

    def attend(self, q, pos, scale):
        """q [nh, hd] at position pos, in 64 bits; also the largest sum of
        |q_i k_i| x scale and the largest |v| that it met, for error bounds."""
        nkv = self.codes.shape[2]
        g = len(q) // nkv
        k = self.codes[0, :pos + 1].astype(np.float64) * self.scales[0][np.arange(pos + 1) // self.block][:, :, None]
        v = self.codes[1, :pos + 1].astype(np.float64) * self.scales[1][np.arange(pos + 1) // self.block][:, :, None]
        out = np.zeros(q.shape, np.float64)
        size = 0.0
        for h in range(len(q)):
            kk, vv = k[:, h // g], v[:, h // g]
            s = kk @ q[h].astype(np.float64) * scale
            size = max(size, float(np.max(np.abs(kk) @ np.abs(q[h].astype(np.float64)))) * scale)
            w = np.exp(s - s.max())
            out[h] = w @ vv / w.sum()
        return out, size, float(np.max(np.abs(v), initial=0.0))
