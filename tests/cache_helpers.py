"""The 8-bit cache and attention over it in numpy, from their definitions: the bytes in binary32, operation by operation, the
attention in binary64 with the tolerance that its arithmetic asks for."""
import numpy as np

from helpers import dev, host, ptr, rng
from tensorrt_amd import capi

TOP = {"int8": np.float32(127), "fp8": np.float32(448)}
TYPE = {"int8": capi.KV_CACHE_INT8, "fp8": capi.KV_CACHE_FP8}


def values(codes, dtype):
    """What bytes stand for before their scale, binary32."""
    if dtype == "int8":
        return codes.view(np.int8).astype(np.float32)
    b = codes.view(np.uint8).astype(np.int32)
    e, m = (b >> 3) & 15, b & 7
    x = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0))
    x = np.where((e == 15) & (m == 7), np.nan, x)
    return np.where(b & 128, -x, x).astype(np.float32)


_CODES = np.arange(127, dtype=np.uint8)
_FP8 = values(_CODES, "fp8")  # 0 .. 448, ascending


def round_codes(y, dtype):
    """Nearest bytes, ties to even, of binary32 values."""
    with np.errstate(invalid="ignore"):
        y = np.clip(y, -TOP[dtype], TOP[dtype]).astype(np.float32)
    if dtype == "int8":
        return np.rint(y).astype(np.int8).view(np.uint8)
    a = np.abs(y).astype(np.float64)
    hi = np.clip(np.searchsorted(_FP8, a), 1, 126)
    lo = hi - 1
    below, above = a - _FP8[lo], _FP8[hi] - a
    code = np.where((below < above) | ((below == above) & (lo % 2 == 0)), lo, hi).astype(np.uint8)
    return code | np.where(np.signbit(y), 128, 0).astype(np.uint8)


class Cache:
    """The pool, its tables, and the model that follows what calls do to it. Unwritten bytes are whatever they happen to be."""

    def __init__(self, dtype, P, H, d, pages, B, max_pages, seed=0, junk=True):
        self.dtype, self.P, self.H, self.d, self.pages, self.B, self.max_pages = dtype, P, H, d, pages, B, max_pages
        r = self.r = rng(seed)
        fill = (lambda s: r.integers(0, 256, s, dtype=np.uint8)) if junk else (lambda s: np.zeros(s, np.uint8))
        self.k, self.v = fill((pages, H, P, d)), fill((pages, H, d, P))
        self.ks, self.vs = (r.uniform(0.5, 2, (pages, H)).astype(np.float32) for _ in range(2))
        self.table = np.full((B, max_pages), -1, np.int32)
        self.lengths = np.zeros(B, np.int32)
        self.free = list(r.permutation(pages))
        self.upload()

    def upload(self):
        self.dk, self.dv, self.dks, self.dvs = dev(self.k), dev(self.v), dev(self.ks), dev(self.vs)
        self.dtable, self.dlengths = dev(self.table), dev(self.lengths)

    def grow(self, new):
        """`new` more tokens of each sequence, with pages for them."""
        self.lengths = self.lengths + np.asarray(new, np.int32)
        for b in range(self.B):
            for i in range(-(-int(self.lengths[b]) // self.P)):
                if self.table[b, i] == -1:
                    self.table[b, i] = self.free.pop()
        self.dtable.copy_(dev(self.table))
        self.dlengths.copy_(dev(self.lengths))

    def described(self, cu, T=None, max_tokens=None):
        """(struct, what it points to)."""
        cu = np.asarray(cu, np.int32)
        dcu = dev(cu)
        n = int(np.diff(cu).max()) if max_tokens is None else max_tokens
        c = capi.KvCache(k=ptr(self.dk), v=ptr(self.dv), k_scale=ptr(self.dks), v_scale=ptr(self.dvs), page_table=ptr(self.dtable),
                         lengths=ptr(self.dlengths), cu_seqlens=ptr(dcu), data_type=TYPE[self.dtype], pages=self.pages, page_tokens=self.P,
                         kv_heads=self.H, d=self.d, B=self.B, max_pages=self.max_pages, max_tokens=n, T=int(cu[-1]) if T is None else T)
        return c, dcu

    def write(self, k, v, cu, T=None, max_tokens=None):
        """The definition, on the model."""
        top = TOP[self.dtype]
        for x, codes, scales, is_v in ((k, self.k, self.ks, False), (v, self.v, self.vs, True)):
            for b in range(self.B):
                all_, end = int(cu[b + 1] - cu[b]), int(self.lengths[b])
                n = min(all_, int(cu[b + 1]) if T is None else T - int(cu[b]), all_ if max_tokens is None else max_tokens)
                begin = end - all_
                tokens = np.arange(begin, begin + n)
                tokens = tokens[(tokens >= 0) & (tokens < self.max_pages * self.P)]
                for block in np.unique(tokens // self.P):
                    page = self.table[b, block]
                    if not 0 <= page < self.pages:
                        continue
                    t = tokens[tokens // self.P == block]
                    new = x[cu[b] + t - begin].astype(np.float32)  # [tokens][H][d]
                    lo, at = t[0] % self.P, t % self.P
                    for h in range(self.H):
                        c = codes[page, h].T if is_v else codes[page, h]
                        old = scales[page, h] if lo > 0 else np.float32(0)
                        a = np.abs(new[:, h]).max()
                        if not np.isfinite(a) or np.isnan(old):
                            scales[page, h] = np.nan
                            c[at] = 0
                            continue
                        limit = old * top
                        scale = old
                        if not limit > 0:
                            scale = a / top
                        else:
                            up = 0
                            while a > limit * np.float32(2.0 ** up):
                                up += 1
                            scale = old * np.float32(2.0 ** up)
                            if up:
                                c[:lo] = round_codes(values(c[:lo].copy(), self.dtype) * np.float32(2.0 ** -up), self.dtype)
                        scales[page, h] = scale
                        c[at] = round_codes(new[:, h] * (np.float32(1) / scale), self.dtype) if scale > 0 else 0

    def check(self):
        """The pool on the GPU against the model, byte by byte."""
        for name in ("k", "v", "ks", "vs"):
            got, want = host(getattr(self, "d" + name)), getattr(self, name)
            same = (got == want) | (np.isnan(got) & np.isnan(want)) if name in ("ks", "vs") else got == want
            assert same.all(), f"{name}: {(~same).sum()} of {same.size} differ, first at {np.argwhere(~same)[:3].tolist()}"

    def codes_of(self, b, which):
        """(values before their scale [tokens][H][d], scales [tokens][H], whether the token is there) of a sequence."""
        n = min(int(self.lengths[b]), self.max_pages * self.P)
        t = np.arange(n)
        page = self.table[b, t // self.P] if n else np.zeros(0, np.int32)
        there = (page >= 0) & (page < self.pages)
        page = np.where(there, page, 0)
        raw = self.k[page, :, t % self.P] if which == "k" else self.v[page, :, :, t % self.P]
        return values(np.ascontiguousarray(raw), self.dtype), (self.ks if which == "k" else self.vs)[page], there


def attention_reference(q, codes_k, scale_k, codes_v, scale_v, visible, scale):
    """One row and head in binary64: (result, tolerance). q [d], codes [keys][d], scales [keys], visible [keys].

    Tolerance. Products of a binary16 and an 8-bit value are exact in binary32, and a score adds d of them, each addition off by at most
    a step of 2^-23 of the running sum (the matrix cores round or cut): d * 2^-23 * sum|q k|. In powers of 2 it is multiplied by scale *
    log2(e) * its page's scale (three roundings), its value scale's logarithm is added (up to 32, within 2^-22 of itself), and the
    maximum subtracted: 6 * 2^-24 * (|s| + 64) more. A weight is off by ln(2) times that, and the exponential by 2^-22 of itself.
    Weights reach the second product as binary16: half a step, 2^-11 of them, or 2^-25 where they are below 2^-14 (the largest is 1 or
    more, so in values that is 2^-25 of the largest value scale for each). The second product's sums and the sum of the weights add up to n
    terms with 2^-23 each; the sums are rescaled and joined, 16 steps more. The result is rounded to binary16."""
    if not visible.any():
        return np.zeros(q.shape), np.zeros(q.shape)
    q = q.astype(np.float64)
    k, v, sk, sv = (np.asarray(x, np.float64)[visible] for x in (codes_k, codes_v, scale_k, scale_v))
    if not (np.isfinite(sk).all() and np.isfinite(sv).all() and np.isfinite(q).all()):
        return np.full(q.shape, np.nan), np.zeros(q.shape)
    n, d = k.shape
    s = (k @ q) * sk * scale
    w = np.exp(s - s.max())
    w /= w.sum()
    out = w @ (v * sv[:, None])
    size = w @ (np.abs(v) * sv[:, None])
    log2e = 1.4426950408889634
    off = (d * 2.0 ** -23 * (np.abs(k) @ np.abs(q)) * sk * scale * log2e + 6 * 2.0 ** -24 * (np.abs(s) * log2e + 64)).max()
    each = np.log(2) * off + 2.0 ** -22
    tol = size * (2.0 ** -11 + 2 * each + 2 * (n + 16) * 2.0 ** -23) + 2.0 ** -25 * sv.max() * np.abs(v).sum(0) + 2.0 ** -11 * np.abs(out) + 2.0 ** -25
    return out, tol * 1.01  # products of these


def assert_within(got, want, tol, what=""):
    got = np.asarray(got, np.float64)
    bad = ~((np.abs(got - want) <= tol) | (np.isnan(got) & np.isnan(want)))
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} outside, worst {np.nanmax(np.abs(got - want) / np.maximum(tol, 1e-30)):.3g} times, at {np.argwhere(bad)[:3].tolist()}"


def visible_keys(at, L, left, right, sinks):
    """Which of L keys the row at `at` sees; left, right: None for all."""
    j = np.arange(L)
    ok = np.ones(L, bool) if right is None else j <= at + right
    if left is not None:
        ok &= (j >= at - left) | (j < sinks)
    return ok
