"""Paged caches, batches and their operators in 64 bits, for tests: e4m3, the cache's order in memory, the formulas."""
import numpy as np

U = 2.0 ** -24                                     # half a step of fp32
LEAST = -120
_CODES = np.arange(127)
# e4m3: 4 exponent bits with bias 7, 3 of the fraction; code 127 is NaN
F8 = np.where(_CODES < 8, _CODES * 2.0 ** -9, (8 + _CODES % 8) * 2.0 ** (_CODES // 8 - 10.0))


def f8_decode(raw):
    raw = np.asarray(raw, np.uint8)
    x = np.append(F8, np.nan)[raw & 127]
    return np.where(raw & 128, -x, x)


def f8_encode(x):
    """Nearest e4m3, ties to the even code; what is not finite: NaN. |x| <= 448."""
    x = np.asarray(x, np.float64)
    a = np.where(np.isfinite(x), np.abs(x), 0)
    lo = np.clip(np.searchsorted(F8, a, side="right") - 1, 0, 125)
    mid = (F8[lo] + F8[lo + 1]) / 2
    code = np.where((a > mid) | ((a == mid) & (lo % 2 == 1)), lo + 1, lo)
    return np.where(np.isfinite(x), code | np.where(np.signbit(x), 128, 0), 127).astype(np.uint8)


def power(top):
    """The least 2^e >= 2^LEAST with top <= 448 * 2^e."""
    m, e = np.frexp(np.asarray(top, np.float64))
    return np.where(top > 0, 2.0 ** np.maximum(LEAST, np.where(m <= 0.875, e - 9, e - 8)), 2.0 ** LEAST)


def pack(k, v):
    """[pages, tokens, kv heads, D] in the cache's order (include/qlinear.h, ql_paged_desc)."""
    P, T, KV, D = k.shape
    u = 16 // k.itemsize
    m = 4 * u
    K = k.reshape(P, T // 16, 16, KV, D // u, u).transpose(0, 3, 1, 4, 2, 5)
    V = v.reshape(P, T // m, u // 4, 4, 4, KV, D // 16, 16).transpose(0, 5, 1, 6, 3, 7, 2, 4)
    return np.ascontiguousarray(K), np.ascontiguousarray(V)


def unpack(K, V):
    P, KV, B, Du, _, u = K.shape
    k = K.transpose(0, 2, 4, 1, 3, 5).reshape(P, B * 16, KV, Du * u)
    v = V.transpose(0, 2, 6, 4, 7, 1, 3, 5).reshape(P, B * 16, KV, Du * u)
    return np.ascontiguousarray(k), np.ascontiguousarray(v)


class Batch:
    """Sequences of (rows, tokens with them) over pages in a shuffled order, `spare` pages more than they need; pad rows behind."""

    def __init__(self, seqs, page, seed=0, spare=2, pad=0):
        g = np.random.default_rng(seed)
        self.seqs, self.page, self.pad = seqs, page, pad
        need = [-(-L // page) for _, L in seqs]
        self.n_page, self.max_pages = sum(need) + spare, max(max(need), 1)
        order, at = g.permutation(self.n_page).astype(np.int32), 0
        self.pages = np.full((len(seqs), self.max_pages), -7, np.int32)      # entries that nothing may follow
        for s, n in enumerate(need):
            self.pages[s, :n] = order[at:at + n]
            at += n
        self.row_start = np.cumsum([0] + [n for n, _ in seqs]).astype(np.int32)
        self.kv_len = np.array([L for _, L in seqs], np.int32)
        self.rows = int(self.row_start[-1])
        self.M = self.rows + pad
        self.max_rows, self.max_len = max(max(n for n, _ in seqs), 1), max(max(L for _, L in seqs), 1)

    def places(self, s):
        """index of each token of sequence s among all pages' tokens"""
        t = np.arange(self.seqs[s][1])
        return self.pages[s][t // self.page].astype(np.int64) * self.page + t % self.page

    def put(self, box, name=""):
        for n in ("row_start", "kv_len", "pages"):
            box.put(name + n, getattr(self, n))

    def desc(self, ql, box, name="", **more):
        kw = {"max_rows": self.max_rows, "max_len": self.max_len, **more}
        return ql.make_batch(box.off(name + "row_start"), box.off(name + "kv_len"), box.off(name + "pages"), len(self.seqs), self.max_pages, **kw)


class Cache:
    """k and v [pages, tokens, kv heads, D]: fp16 bits, or e4m3 codes with a scale for 16 tokens of a head."""

    def __init__(self, f8, n_page, page, KV, D, seed=0, empty=False):
        g = np.random.default_rng([seed, 77])
        self.f8, self.KV, self.D, self.page, self.n_page = f8, KV, D, page, n_page
        shape, groups = (n_page, page, KV, D), (n_page, page // 16, KV)
        self.scale = {}
        for n in "kv":
            x = g.standard_normal(shape)
            if empty:                                                            # what nothing was appended to may hold anything
                x = np.full(shape, 127, np.uint8) if f8 else np.full(shape, np.nan, np.float16)
                if f8:
                    self.scale[n] = np.full(groups, np.nan, np.float32)
            elif f8:
                p = power(np.abs(x).reshape(n_page, page // 16, 16, KV, D).max((2, 4)))
                self.scale[n] = p.astype(np.float32)
                x = f8_encode(x / np.repeat(p, 16, 1)[..., None])
            else:
                x = x.astype(np.float16)
            setattr(self, n, x)

    def values(self, n):
        """[tokens of all pages, kv heads, D] in 64 bits"""
        x = getattr(self, n)
        if self.f8:
            with np.errstate(invalid="ignore"):
                x = f8_decode(x) * np.repeat(self.scale[n].astype(np.float64), 16, 1)[..., None]
        return x.astype(np.float64).reshape(-1, self.KV, self.D)

    def put(self, box, name=""):
        K, V = pack(self.k, self.v)
        self.name = name
        box.put(name + "K", K), box.put(name + "V", V)
        if self.f8:
            for n in "kv":
                box.put(name + n + "s", self.scale[n].transpose(0, 2, 1))

    def desc(self, ql, box):
        n = self.name
        more = dict(k_scale_off=box.off(n + "ks"), v_scale_off=box.off(n + "vs")) if self.f8 else {}
        return ql.make_paged(box.off(n + "K"), box.off(n + "V"), self.n_page, self.page, self.KV, self.D,
                             cache_dtype=ql.DTYPE_F8 if self.f8 else ql.DTYPE_F16, **more)

    def read(self, box):
        """another cache, with what the device holds now"""
        c = Cache.__new__(Cache)
        c.f8, c.KV, c.D, c.page, c.n_page, c.name = self.f8, self.KV, self.D, self.page, self.n_page, self.name
        c.k, c.v = unpack(box.get(self.name + "K"), box.get(self.name + "V"))
        c.scale = {n: box.get(self.name + n + "s").transpose(0, 2, 1).copy() for n in "kv"} if self.f8 else {}
        return c


def attention(q, cache, batch):
    """(out, tolerance of fp32 results, sum of p |v|) in 64 bits; rows of padding are NaN."""
    M, H, D = q.shape
    q = q.astype(np.float64)
    KV = cache.KV
    G = H // KV
    out, tol, size = (np.full(q.shape, np.nan) for _ in range(3))
    k_all, v_all = cache.values("k"), cache.values("v")
    for s, (n, L) in enumerate(batch.seqs):
        if n == 0:
            continue
        at, r0 = batch.places(s), int(batch.row_start[s])
        for kv in range(KV):
            k, v = k_all[at, kv], v_all[at, kv]
            h = slice(kv * G, (kv + 1) * G)
            x = q[r0:r0 + n, h].reshape(n * G, D)
            seen = np.repeat(np.arange(L)[None] <= np.arange(L - n, L)[:, None], G, 0)
            with np.errstate(all="ignore"):
                sc = np.where(seen, x @ k.T / np.sqrt(D), -np.inf)
                top = sc.max(1, keepdims=True)
                p = np.exp(sc - np.where(top == -np.inf, 0, top))
                p = np.where(seen, p, 0)
                total = p.sum(1, keepdims=True)
                vz = np.where(seen.any(0)[:, None], v, 0)
                poisoned = ~np.isfinite(vz).all()
                if poisoned:                                                     # what a row does not see adds nothing to it
                    o = np.stack([(p[r][seen[r]][:, None] * v[seen[r]]).sum(0) for r in range(n * G)])
                else:
                    o = p @ vz
                o = np.where(total == 0, 0, o / total)
                # q's parts carry 2^-22 of its row's largest, fp32 sums of D products D u of the products' sizes, the exponential's argument
                # and its own value 2^-22 and 2^-22 of the score's size; the errors of two scores move a weight
                a = np.where(seen, np.abs(x) @ np.abs(k).T / np.sqrt(D), 0)
                reach = np.abs(x).max(1, keepdims=True) * np.abs(k).sum(1) / np.sqrt(D) * 2.0 ** -22
                e = np.where(seen, (D + 8) * U * a + reach + 2.0 ** -21 * (np.abs(np.where(seen, sc, 0)) + 1), 0)
                e = np.nan_to_num(e, nan=0, posinf=0)
                pv = p @ np.abs(np.nan_to_num(vz, nan=0, posinf=0, neginf=0)) / np.where(total > 0, total, 1)
                big = np.abs(np.nan_to_num(vz, nan=0, posinf=0, neginf=0)).max(0)
                w = p / np.where(total > 0, total, 1)
                # each weight off by 2 e (its own and the sum's); P's parts 2^-22 of a weight down to 2^-33 of the largest; sums of L / 32 terms
                t = 2 * (w * e) @ np.abs(np.nan_to_num(vz, nan=0, posinf=0, neginf=0)) + 2 * (w * e).sum(1, keepdims=True) * pv + \
                    (2.0 ** -20 + (L / 32 + 64) * U) * pv + L * 2.0 ** -33 * big
            out[r0:r0 + n, h] = o.reshape(n, G, D)
            tol[r0:r0 + n, h] = t.reshape(n, G, D)
            size[r0:r0 + n, h] = pv.reshape(n, G, D)
    return out, tol, size


def turned(x, pos, norm, eps, theta, rot, interleaved):
    """(values, tolerance of fp32's) of heads x [M, heads, D] in 64 bits"""
    x = x.astype(np.float64)
    D = x.shape[-1]
    if norm is not None:
        x = x / np.sqrt((x ** 2).mean(-1, keepdims=True) + eps) * norm.astype(np.float64)
    t = pos[:, None] * theta ** (-2.0 * np.arange(rot // 2) / rot)
    c, s = np.cos(t)[:, None], np.sin(t)[:, None]
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    y, size = x.copy(), np.abs(x)
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    both = size[..., a] + size[..., b]
    size[..., a] = size[..., b] = both
    # the norm's sum of D squares, its root, quotient and two products; the table's rounding, two products and their sum
    return y, ((D / 2 + 8 if norm is not None else 0) + 6) * U * size
