"""What the tests of the serving operators share: device buffers without torch, a page book kept in Python lists, and attention in
64 bits."""
import ctypes

import numpy as np

from conftest import bf16_bits, bf16_vals

BF16_HALF_STEP, F32_HALF_STEP = 2.0 ** -8, 2.0 ** -24


def hip():
    """The HIP runtime that libq3asr.so has loaded."""
    with open("/proc/self/maps") as f:
        paths = sorted({line.split()[-1] for line in f if "libamdhip64" in line})
    own = [p for p in paths if "/torch/" not in p] or paths
    h = ctypes.CDLL(own[0])
    P, V = ctypes.POINTER, ctypes.c_void_p
    h.hipMalloc.argtypes = [P(V), ctypes.c_size_t]
    h.hipMemcpy.argtypes = [V, V, ctypes.c_size_t, ctypes.c_int]
    h.hipFree.argtypes = [V]
    h.hipStreamCreate.argtypes = [P(V)]
    h.hipStreamSynchronize.argtypes = [V]
    h.hipStreamDestroy.argtypes = [V]
    h.hipStreamBeginCapture.argtypes = [V, ctypes.c_int]
    h.hipStreamEndCapture.argtypes = [V, P(V)]
    h.hipGraphInstantiate.argtypes = [P(V), V, V, V, ctypes.c_size_t]
    h.hipGraphLaunch.argtypes = [V, V]
    h.hipGraphExecDestroy.argtypes = [V]
    h.hipGraphDestroy.argtypes = [V]
    return h


class Device:
    """Arrays in device memory, freed together."""

    def __init__(self):
        self.h, self.held, self.streams = hip(), [], []

    def raw(self, nbytes):
        p = ctypes.c_void_p()
        assert self.h.hipMalloc(ctypes.byref(p), max(int(nbytes), 16)) == 0
        self.held.append(p)
        return p.value

    def put(self, a, at=None):
        a = np.ascontiguousarray(a)
        at = self.raw(a.nbytes) if at is None else at
        assert self.h.hipMemcpy(at, a.ctypes.data, a.nbytes, 1) == 0
        return at

    def get(self, at, shape, dtype):
        a = np.empty(shape, dtype)
        assert self.h.hipMemcpy(a.ctypes.data, at, a.nbytes, 2) == 0
        return a

    def stream(self):
        s = ctypes.c_void_p()
        assert self.h.hipStreamCreate(ctypes.byref(s)) == 0
        self.streams.append(s)
        return s.value

    def wait(self, s):
        assert self.h.hipStreamSynchronize(s) == 0

    def capture(self, s, calls):
        """A graph of what `calls` enqueues on s."""
        g, x = ctypes.c_void_p(), ctypes.c_void_p()
        assert self.h.hipStreamBeginCapture(s, 2) == 0   # relaxed
        calls()
        assert self.h.hipStreamEndCapture(s, ctypes.byref(g)) == 0
        assert self.h.hipGraphInstantiate(ctypes.byref(x), g, None, None, 0) == 0
        assert self.h.hipGraphDestroy(g) == 0
        return x

    def __enter__(self):
        return self

    def __exit__(self, *a):
        self.h.hipDeviceSynchronize()
        for s in self.streams:
            self.h.hipStreamDestroy(s)
        for p in self.held:
            self.h.hipFree(p)


class Book:
    """A paged cache as Python lists, one call after the other by the documented rules; contents as numpy arrays."""

    def __init__(self, k, v, seqs, width):
        self.k, self.v = k.copy(), v.copy()          # [layers][pages][heads][page][dim]
        self.pg, self.width = k.shape[3], width
        self.refs = [0] * k.shape[1]
        self.tables, self.lens = [[] for _ in range(seqs)], [0] * seqs

    def fork(self, dst, src):
        old = [(list(self.tables[q]), self.lens[q]) if q >= 0 else ([], 0) for q in src]
        for d, (t, n) in zip(dst, old):
            for p in self.tables[d]:
                self.refs[p] -= 1
            for p in t:
                self.refs[p] += 1
            self.tables[d], self.lens[d] = t, n

    def reserve(self, seqs, tokens):
        free = [p for p, r in enumerate(self.refs) if r == 0][::-1]
        part = {s: self.tables[s][-1] for s, a in zip(seqs, tokens) if a and self.lens[s] % self.pg}
        holders = {}
        for s in seqs:
            if s in part:
                holders.setdefault(part[s], []).append(s)
        before = list(self.refs)
        for s, add in zip(seqs, tokens):
            if s in part:
                p, fill = part[s], self.lens[s] % self.pg
                keeps = len(holders[p]) == before[p] and holders[p][0] == s
                if before[p] > 1 and not keeps:
                    to = free.pop()
                    for pool in (self.k, self.v):
                        pool[:, to, :, :fill] = pool[:, p, :, :fill]
                    self.refs[p] -= 1
                    self.refs[to] = 1
                    self.tables[s][-1] = to
            self.lens[s] += add
            while len(self.tables[s]) * self.pg < self.lens[s]:
                self.tables[s].append(free.pop())
                self.refs[self.tables[s][-1]] = 1

    def compact(self):
        n = sum(r > 0 for r in self.refs)
        gaps = [p for p in range(n) if not self.refs[p]]
        to = dict(zip([p for p in range(n, len(self.refs)) if self.refs[p]], gaps))
        for p, g in to.items():
            for pool in (self.k, self.v):
                pool[:, g] = pool[:, p]
            self.refs[g], self.refs[p] = self.refs[p], 0
        self.tables = [[to.get(p, p) for p in t] for t in self.tables]
        return n

    def write(self, layer, k_rows, v_rows, seqs, cu):
        for i, s in enumerate(seqs):
            for r in range(cu[i], cu[i + 1]):
                pos = self.lens[s] - (cu[i + 1] - r)
                p = self.tables[s][pos // self.pg]
                self.k[layer, p, :, pos % self.pg] = k_rows[r].reshape(self.k.shape[2], -1)
                self.v[layer, p, :, pos % self.pg] = v_rows[r].reshape(self.k.shape[2], -1)

    def table(self):
        return np.array([t + [-1] * (self.width - len(t)) for t in self.tables], np.int32).reshape(-1, self.width)

    def keys(self, layer, s):
        """K and V values of a sequence: [heads][len][dim], 64 bits."""
        out = []
        for pool in (self.k, self.v):
            x = bf16_vals(pool[layer, self.tables[s]]).astype(np.float64) if self.tables[s] else np.zeros((0,) + pool.shape[2:])
            out.append(x.transpose(1, 0, 2, 3).reshape(pool.shape[2], -1, pool.shape[4])[:, :self.lens[s]])
        return out


class Cache:
    """A PagedKVCache on the device beside the book of the same contents."""

    def __init__(self, dev, model, seqs, width, pages, layers=1, heads=2, dim=128, pg=16, seed=0, poison=False):
        from q3asr import PagedKVCache
        rng = np.random.default_rng(seed)
        shape = (layers, pages, heads, pg, dim)
        self.dev, self.shape, self.seqs, self.width = dev, shape, seqs, width
        if poison:   # whatever was not written holds NaN
            k = v = np.full(shape, 0x7FC1, np.uint16)
        else:
            k, v = (bf16_bits(rng.standard_normal(shape)) for _ in range(2))
        self.book = Book(k, v, seqs, width)
        self.at = {"k": dev.put(k), "v": dev.put(v), "table": dev.raw(4 * seqs * width), "lens": dev.raw(4 * seqs), "refs": dev.raw(4 * pages),
                   "status": dev.raw(16)}
        self.c = PagedKVCache(model, layers=layers, pages=pages, kv_heads=heads, head_dim=dim, page_tokens=pg, max_seqs=seqs,
                              max_seq_pages=width, **self.at)
        n = self.c.workspace_bytes()
        self.c.set_workspace(dev.raw(n), n)
        self.c.reset()

    def put(self):
        """The book's state onto the device."""
        self.dev.put(self.book.table(), self.at["table"])
        self.dev.put(np.array(self.book.lens, np.int32), self.at["lens"])
        self.dev.put(np.array(self.book.refs, np.int32), self.at["refs"])

    def ints(self, v):
        return self.dev.put(np.asarray(v, np.int32))

    def fork(self, dst, src, stream=None):
        self.c.fork(self.ints(dst), self.ints(src), len(dst), stream)
        self.book.fork(dst, src)

    def reserve(self, seqs, tokens, stream=None):
        self.c.reserve(self.ints(seqs), self.ints(tokens), len(seqs), stream)
        self.book.reserve(seqs, tokens)

    def free(self, seqs, stream=None):
        self.c.free(self.ints(seqs), len(seqs), stream)
        self.book.fork(seqs, [-1] * len(seqs))

    def compact(self, stream=None):
        self.c.compact(stream)
        return self.book.compact()

    def state(self):
        d, (layers, pages, heads, pg, dim) = self.dev, self.shape
        return (d.get(self.at["table"], (self.seqs, self.width), np.int32), d.get(self.at["lens"], self.seqs, np.int32),
                d.get(self.at["refs"], pages, np.int32), d.get(self.at["k"], self.shape, np.uint16), d.get(self.at["v"], self.shape, np.uint16))

    def check(self):
        table, lens, refs, k, v = self.state()
        assert lens.tolist() == self.book.lens
        assert refs.tolist() == self.book.refs
        assert np.array_equal(table, self.book.table())
        assert np.array_equal(k, self.book.k) and np.array_equal(v, self.book.v)


def attention64(q, k, v, lens, rows, heads, scale):
    """One sequence: q [rows][heads][dim] at its last positions, k / v [kv][len][dim], all 64 bits.  Returns the rows' outputs,
    logarithms of their sums, and what their rounding errors are measured by: sum_j p_j |v_j| and the score error bound."""
    kv, n, d = k.shape
    out, lse = np.zeros((rows, heads, d)), np.full((rows, heads), -np.inf)
    size, slack = np.zeros((rows, heads, d)), np.zeros((rows, heads))
    for t in range(rows):
        seen = lens - rows + t + 1
        if seen <= 0:
            continue
        for h in range(heads):
            kk, vv = k[h * kv // heads, :seen], v[h * kv // heads, :seen]
            s = kk @ q[t, h] * scale
            m = s.max()
            p = np.exp(s - m)
            lse[t, h] = m + np.log(p.sum())
            p /= p.sum()
            out[t, h], size[t, h] = p @ vv, p @ np.abs(vv)
            # fp32 sum of d exact products, the scaling, and exp2 of an argument of that size
            slack[t, h] = (d + 4) * F32_HALF_STEP * 2 * (np.abs(kk) @ np.abs(q[t, h])).max() * abs(scale) + 8 * F32_HALF_STEP
    return out, lse, size, slack


def attention_bounds(out, size, slack, keys):
    """Largest error of a bf16 result: its own rounding; the probabilities' rounding to bf16 in the sum; the scores' errors in
    numerator and denominator; fp32 sums over the keys (in parts, so their number bounds it from above)."""
    return BF16_HALF_STEP * np.abs(out) * (1 + 1e-3) + (BF16_HALF_STEP + 2 * slack[..., None] + 2 * (keys + 64) * F32_HALF_STEP) * size + 1e-30
