"""The paged key/value cache and its attention in plain 64-bit arithmetic, and a small cache on the device to compare with."""
import numpy as np
import torch

CODES = {"int8": 127.0, "fp8": 448.0}


def rotated(x, cos, sin, rotary):
    """x [rows, heads, D] fp16 -> fp16; products and sums rounded to 32 bits one by one."""
    y, h = x.copy(), rotary // 2
    a, b = x[..., :h].astype(np.float32), x[..., h:rotary].astype(np.float32)
    c, s = cos[:, None], sin[:, None]
    with np.errstate(over="ignore", invalid="ignore"):
        y[..., :h] = (a * c - b * s).astype(np.float16)
        y[..., h:rotary] = (b * c + a * s).astype(np.float16)
    return y


def quantised(x, fmt):
    """Codes (as bytes) and fp16 scales of fp16 rows [..., D]."""
    x = x.astype(np.float64)
    most = np.abs(x).max(axis=-1)
    good = np.isfinite(most)
    want = np.where(good, most, 0.0) / CODES[fmt]
    grid = np.exp2(np.maximum(np.floor(np.log2(np.maximum(want, 2.0 ** -60))) - 10, -24))   # the distance of neighbours in fp16
    scale = np.ceil(want / grid) * grid
    scale = np.where(scale * CODES[fmt] > 65504, scale - grid, scale)   # (the largest fp16 value reads back as a finite one)
    scale = np.where(want == 0, 1.0, scale)
    y = np.where(good[..., None], np.nan_to_num(x, posinf=0, neginf=0), 0.0) / scale[..., None]
    if fmt == "int8":
        codes = np.rint(y).astype(np.int8).view(np.uint8)
    else:
        codes = torch.from_numpy(y.astype(np.float32)).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    return codes, np.where(good, scale, np.nan).astype(np.float16)


def code_values(codes, fmt):
    if fmt == "int8":
        return codes.view(np.int8).astype(np.float64)
    return torch.from_numpy(np.ascontiguousarray(codes)).view(torch.float8_e4m3fn).double().numpy()


def attend(q, k, v, positions, scale, window, sinks):
    """One head: q [n, D], k and v [length, D] in 64 bits; also what an error bound needs.  Hidden keys are not touched."""
    n, D = q.shape
    out, spread, most, steep = np.zeros((n, D)), np.zeros((n, D)), np.zeros(n), np.zeros(n)
    for i, p in enumerate(positions):
        key = np.arange(min(p + 1, len(k)))
        if window:
            key = key[(key > p - window) | (key < sinks)]
        if not len(key):
            continue
        with np.errstate(invalid="ignore", over="ignore"):
            s = scale * (k[key] @ q[i])
            w = np.exp(s - s.max())
            w /= w.sum()
            out[i] = w @ v[key]
            spread[i] = w @ np.abs(v[key])
            # (rows that see what is not finite are computed with weights of 32 bits; a key at an infinite distance has the weight 0 without an error)
            most[i] = np.abs(v[key], where=np.isfinite(v[key]), out=np.zeros_like(v[key])).max()
            far = np.abs(k[key]) @ np.abs(q[i])
            steep[i] = scale * np.where(np.isfinite(far), far, 0).max()
    return out, spread, most, steep


def attention_bound(out, spread, most, steep, length, D):
    """How far an fp16 result of 32-bit sums may be off: the result's own rounding (half a step, 2^-11); the rounding of each weight to fp16
    for the second product, 2^-11 of it, or 2^-25 of the largest one where it is subnormal; and the error of a score, which moves its weight and
    the sum of the weights: sums of D products of 32 bits (D 2^-23 of the sum of magnitudes, whichever way they are added), the
    subtraction of the maximum and the exponential's own error of 2^-21."""
    score = 2.0 ** -21 + steep * (D + 4) * 2.0 ** -23
    return 2.0 ** -11 * np.abs(out) + (2.0 ** -11 + 2 * score + length * 2.0 ** -24)[..., None] * spread + (length * 2.0 ** -25 * most)[..., None] + 2.0 ** -24


class Cache:
    """A cache on the device with its sequences' pages scattered, pages beyond them and cells behind each end holding NaNs, and its contents on the host."""

    def __init__(self, nnb, ctx, fmt, lengths, kv_heads, D, page, seed, extra_pages=2, first_page=0, fill=True):
        self.nnb, self.ctx, self.fmt, self.kv_heads, self.D, self.page = nnb, ctx, fmt, kv_heads, D, page
        rng = np.random.default_rng(seed)
        need = [-(-n // page) for n in lengths]
        self.pages = sum(need) + extra_pages
        order = rng.permutation(self.pages)
        self.table = np.full((max(1, len(lengths)), max(need + [1]) + 1), -7, np.int32)
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = order[at:at + n]
            at += n
        shape = (self.pages, kv_heads, page, D)
        self.lengths = lengths
        self.host, self.dev = {}, {}
        for name in "kv":
            rows = rng.standard_normal(shape).astype(np.float16)
            if fmt == "fp16":
                codes, scale = rows.view(np.uint16), None
            else:
                codes, scale = quantised(rows, fmt)
            if fill:
                stale = np.ones((self.pages, page), bool)
                for i, n in enumerate(lengths):
                    for p in range(n):
                        stale[self.table[i, p // page], p % page] = False
                stale = np.repeat(stale[:, None], kv_heads, axis=1)
                if fmt == "fp16":
                    codes[stale] = 0x7E00
                else:
                    scale[stale] = np.float16(np.nan)
            self.host[name], self.host[name + "_scale"] = codes, scale
            self.dev[name] = ctx.upload(codes)
            self.dev[name + "_scale"] = None if scale is None else ctx.upload(scale.view(np.uint16))
        self.handle = ctx.kv_cache(fmt, self.pages, page, kv_heads, D, self.dev["k"], self.dev["v"], self.dev["k_scale"], self.dev["v_scale"])
        self.kept = []

    def batch(self, new, lengths=None, extra_rows=0, max_new=None, max_len=None, table=None, row_start=None):
        lengths = self.lengths if lengths is None else lengths
        start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32) if row_start is None else np.asarray(row_start, np.int32)
        table = self.table if table is None else table
        up = [self.ctx.upload(np.ascontiguousarray(a, np.int32)) for a in (start, np.asarray(lengths, np.int32), table)]
        self.kept += up
        return self.nnb.KVBatch(len(lengths), int(start[-1]) + extra_rows, max_new or max(1, max(new)), max_len or table.shape[1] * self.page, table.shape[1], *up)

    def sequence(self, name, i, length):
        """[length, kv_heads, D] in 64 bits, as the host has it."""
        codes, scale = self.host[name], self.host[name + "_scale"]
        p = np.arange(length)
        page, slot = self.table[i, p // self.page], p % self.page
        if self.fmt == "fp16":
            return codes[page, :, slot].view(np.float16).astype(np.float64)
        return code_values(codes[page, :, slot], self.fmt) * scale[page, :, slot].astype(np.float64)[..., None]

    def read_back(self):
        """The device's pages (and scales) as the host would have them."""
        got = {}
        for name in "kv":
            got[name] = self.ctx.download(self.dev[name], self.host[name].shape, self.host[name].dtype)
            if self.fmt != "fp16":
                got[name + "_scale"] = self.ctx.download(self.dev[name + "_scale"], self.host[name + "_scale"].shape, np.uint16)
        return got

    def close(self):
        self.ctx.sync()
        self.handle.close()
        for b in [*self.kept, *(d for d in self.dev.values() if d)]:
            self.ctx.free(b)
