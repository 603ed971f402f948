"""8-bit integer products against whole-number arithmetic in 64 bits, through the C ABI on device buffers."""
import numpy as np
import pytest

from conftest import bf16_bits, bf16_vals
from serving_kit import BF16_HALF_STEP, F32_HALF_STEP, Device

pytestmark = pytest.mark.gpu


def _quantize64(x):
    """Scales and whole numbers of rows, by the operator's definition."""
    x = x.astype(np.float32)
    with np.errstate(all="ignore"):
        amax = np.abs(x).max(1)
        scale = (amax / np.float32(127)).astype(np.float32)
        bad = ~np.isfinite(amax)
        safe = np.where(bad | (scale == 0), 1, scale).astype(np.float64)
        q = np.clip(np.rint(np.where(bad[:, None], 0, x.astype(np.float64)) / safe[:, None]), -127, 127)
        q[(scale == 0) | bad] = 0
        scale[bad] = np.nan
    return scale, q.astype(np.int64)


def _rows(rng, m, k, kind):
    x = rng.standard_normal((m, k)) * np.exp(rng.standard_normal((m, 1)))
    x[:, rng.random(k) < 0.02] *= 15
    return x.astype(np.float32) if kind == "f32" else bf16_vals(bf16_bits(x))


def _put_rows(dev, x, ld, kind):
    """x with a row stride of ld values; what lies between the rows is NaN."""
    wide = np.full((x.shape[0], ld), np.nan, np.float32)
    wide[:, :x.shape[1]] = x
    return dev.put(wide if kind == "f32" else bf16_bits(wide))


def _weights(rng, n, k):
    """Weights with rows padded to 16, what lies behind K set to 55 (it must not count)."""
    ldw = (k + 15) // 16 * 16
    w = np.full((n, ldw), 55, np.int8)
    w[:, :k] = rng.integers(-127, 128, (n, k))
    return w, ldw, (rng.random(n) * 0.01 + 1e-4).astype(np.float32)


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("m,k,pad", [(1, 1, 0), (3, 15, 1), (5, 16, 0), (4, 17, 8), (70, 1003, 5), (33, 2048, 0), (2, 6144, 24), (9, 4100, 4),
                                     (3, 9003, 0), (1100, 300, 3), (1030, 5000, 0), (1030, 7001, 1)])
def test_quantize_rows_is_exact(tiny_model, m, k, pad, kind):
    from q3asr import quantize_rows
    rng = np.random.default_rng(m * 31 + k)
    x = _rows(rng, m, k, kind)
    ldq = (k + 15) // 16 * 16 + 16
    with Device() as dev:
        q, s = dev.put(np.full((m, ldq), 99, np.int8)), dev.raw(4 * m)
        quantize_rows(tiny_model[0], _put_rows(dev, x, k + pad, kind), m, k, q, s, x_dtype=kind, ldx=k + pad, ldq=ldq)
        got, scale = dev.get(q, (m, ldq), np.int8), dev.get(s, m, np.float32)
    want_s, want_q = _quantize64(x)
    k16 = (k + 15) // 16 * 16
    assert np.array_equal(scale, want_s)
    assert np.array_equal(got[:, :k], want_q)
    assert (got[:, k:k16] == 0).all() and (got[:, k16:] == 99).all()   # padding is zero, the rest is left alone


def test_quantize_rows_at_the_borders(tiny_model):
    """Rows of zeros, one infinity, one NaN, denormals, the largest numbers; quotients at and beside the middle of two whole numbers."""
    from q3asr import quantize_rows
    f = np.float32
    k = 512
    rows = [np.zeros(k, f), np.ones(k, f), np.ones(k, f), np.full(k, 1e-44, f), np.linspace(-3e-41, 3e-41, k).astype(f),
            np.linspace(-3.4e38, 3.4e38, k).astype(f), np.linspace(-2e-36, 2e-36, k).astype(f), np.linspace(-1e-30, 1e-30, k).astype(f)]
    rows[1][7], rows[2][9] = np.inf, np.nan
    ties = np.zeros(k, f)
    ties[0] = 127.0                       # scale 1: halves are ties
    ties[1:250] = np.arange(249) - 124 + f(0.5)
    ties[250:499] = np.nextafter(np.arange(249, dtype=f) - 124 + f(0.5), f(1e9))
    rows.append(ties)
    for seed in range(6):                 # values one step around (n + 1/2) * scale for awkward scales
        rng = np.random.default_rng(seed)
        amax = f(rng.random() + 0.5)
        s = f(amax / f(127))
        mid = ((rng.integers(-126, 126, k) + 0.5) * float(s)).astype(f)
        r = np.where(rng.random(k) < 0.5, np.nextafter(mid, f(9)), mid).astype(f)
        r[0] = amax
        rows.append(r)
    x = np.stack(rows)
    with Device() as dev:
        q, s = dev.raw(x.size), dev.raw(4 * len(rows))
        quantize_rows(tiny_model[0], dev.put(x), len(rows), k, q, s, x_dtype="f32")
        got, scale = dev.get(q, x.shape, np.int8), dev.get(s, len(rows), np.float32)
    want_s, want_q = _quantize64(x)
    assert np.array_equal(scale, want_s, equal_nan=True)
    assert np.array_equal(got, want_q)
    assert np.isnan(scale[1]) and np.isnan(scale[2]) and scale[0] == 0


@pytest.mark.parametrize("rows", [128, 1152])
def test_quantize_every_ratio_of_bf16_values(tiny_model, rows):
    """Every pair of bf16 mantissas as value and maximum of a row, the value smaller by up to 2^9, either sign: all quotients that lie
    half way between two whole numbers before the scale is rounded, and all next to them; with the product's own rounding as well."""
    from q3asr import Int8Linear, quantize_rows
    a = (np.arange(256)[None, :] / 2.0 ** np.arange(10)[:, None]).reshape(-1)
    a = np.concatenate([a, -a])
    tops = np.arange(128, 256, dtype=np.float64)
    x = np.where(np.abs(a) <= tops[:, None], a, 0)
    x[:, 0] = tops
    x = np.concatenate([x * 2.0 ** e for e in range(-40, -40 + 10 * (rows // 128), 10)]).astype(np.float32)
    assert np.array_equal(bf16_vals(bf16_bits(x)), x)
    m, k = x.shape
    with Device() as dev:
        model = tiny_model[0]
        q, s, at = dev.raw(m * k), dev.raw(4 * m), dev.put(bf16_bits(x))
        quantize_rows(model, at, m, k, q, s)
        got, scale = dev.get(q, (m, k), np.int8), dev.get(s, m, np.float32)
        want_s, want_q = _quantize64(x)
        assert np.array_equal(scale, want_s) and np.array_equal(got, want_q)
        lin = Int8Linear(model, q, s, m, k)          # few rows are rounded inside the product
        o, ref, ws = dev.raw(4 * m), dev.raw(4 * m), lin.workspace_bytes(1)
        for row in range(0, m, 37):
            lin(at + 2 * k * row, 1, o, out_dtype="f32", workspace=(dev.raw(ws), ws))
            lin.matmul(q + k * row, s + 4 * row, 1, ref, out_dtype="f32")
            assert np.array_equal(dev.get(o, m, np.float32), dev.get(ref, m, np.float32)), row


SHAPES = [(1, 1, 1), (1, 4096, 2048), (2, 33, 100), (3, 2048, 6144), (4, 64, 33), (5, 70, 1003), (8, 256, 512), (16, 1000, 784),
          (17, 31, 48), (31, 515, 2080), (64, 64, 128), (65, 127, 129), (130, 2048, 4096), (200, 320, 6000), (333, 1027, 1003), (700, 769, 300),
          (2100, 2304, 256), (300, 12288, 96), (1000, 1500, 200), (3100, 4001, 130), (3100, 4000, 640), (40, 40000, 64), (6, 96, 6200), (2, 50, 13000)]


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("x,out,bias", [("bf16", "bf16", False), ("f32", "f32", True)])
def test_linear_matches_whole_numbers(tiny_model, m, n, k, x, out, bias):
    from q3asr import Int8Linear
    rng = np.random.default_rng(m + 7 * n + 11 * k)
    xs = _rows(rng, m, k, x)
    w, ldw, sw = _weights(rng, n, k)
    b = rng.standard_normal(n).astype(np.float32) if bias else None
    ldo = n + (3 if bias else 0)
    dt = np.float32 if out == "f32" else np.uint16
    fill = np.full((m, ldo), 7, dt)
    with Device() as dev:
        lin = Int8Linear(tiny_model[0], dev.put(w), dev.put(sw), n, k, ldw=ldw, bias=dev.put(b) if bias else None)
        ws = lin.workspace_bytes(m)
        o = dev.put(fill)
        lin(_put_rows(dev, xs, k + 1, x), m, o, x_dtype=x, ldx=k + 1, out_dtype=out, ldo=ldo, workspace=(dev.raw(ws), ws))
        got = dev.get(o, (m, ldo), dt)
    assert (got[:, n:] == 7).all()                       # what lies between the rows is left alone
    got = (got if out == "f32" else bf16_vals(got))[:, :n].astype(np.float64)
    s, q = _quantize64(xs)
    prod = (q.astype(np.float64) @ w[:, :k].astype(np.float64).T) * s.astype(np.float64)[:, None] * sw.astype(np.float64)   # sums below 2^53
    want = prod if b is None else prod + b
    # the sum to fp32, two products, the bias, then the result's type
    tol = 3.01 * F32_HALF_STEP * np.abs(prod) + 1.01 * F32_HALF_STEP * np.abs(want)
    if out == "bf16":
        tol = tol * 1.01 + BF16_HALF_STEP * np.abs(want)
    assert (np.abs(got - want) <= tol + 1e-37).all()


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("m,ks", [(1, range(7, 26)), (3, range(513, 523)), (5, range(2094, 2103)), (6, (1363, 1364, 4001)),
                                  (8, (2041, 2048)), (13, (3, 7, 8)), (16, range(1009, 1026)), (40, range(130, 139))])
def test_linear_of_any_length_and_alignment(tiny_model, m, ks, kind):
    """Every length against whole pieces of 8 values; activations and outputs begin one value behind an aligned address."""
    from q3asr import Int8Linear
    rng = np.random.default_rng(m)
    n, size, dt = 90, 4 if kind == "f32" else 2, np.float32 if kind == "f32" else np.uint16
    for k in ks:
        xs = _rows(rng, m, k, kind)
        w, ldw, sw = _weights(rng, n, k)
        with Device() as dev:
            lin = Int8Linear(tiny_model[0], dev.put(w), dev.put(sw), n, k, ldw=ldw)
            ws, o = lin.workspace_bytes(m), dev.put(np.full(m * n + 2, 7, dt))
            flat = np.full(m * k + 2, np.nan, np.float32)
            flat[1:-1] = xs.reshape(-1)
            x = dev.put(flat if kind == "f32" else bf16_bits(flat))
            lin(x + size, m, o + size, x_dtype=kind, out_dtype=kind, workspace=(dev.raw(ws), ws))
            got = dev.get(o, m * n + 2, dt)
        assert got[0] == 7 and got[-1] == 7
        got = (got if kind == "f32" else bf16_vals(got))[1:-1].reshape(m, n).astype(np.float64)
        s, q = _quantize64(xs)
        want = (q.astype(np.float64) @ w[:, :k].astype(np.float64).T) * s.astype(np.float64)[:, None] * sw.astype(np.float64)
        tol = 3.01 * F32_HALF_STEP * np.abs(want) + (1.01 * BF16_HALF_STEP * np.abs(want) if kind == "bf16" else 0)
        assert (np.abs(got - want) <= tol + 1e-37).all(), k


@pytest.mark.parametrize("m,n,k", [(1, 40, 64), (6, 300, 4096), (70, 130, 1024), (260, 300, 2048), (1000, 768, 131056 // 16), (2, 3, 131056)])
def test_matmul_equals_linear_and_extremes(tiny_model, m, n, k):
    """quantize + matmul gives linear's bits; -128 (which quantize never makes) and rows of +-127 sum without overflow."""
    from q3asr import Int8Linear, quantize_rows
    rng = np.random.default_rng(k)
    k = k // 16 * 16
    xs = _rows(rng, m, k, "bf16")
    w, ldw, sw = _weights(rng, n, k)
    w[0], w[-1] = 127, -128
    a = rng.integers(-128, 128, (m, k)).astype(np.int8)
    a[0], a[-1] = -128, 127
    sa = (rng.random(m) + 0.5).astype(np.float32)
    with Device() as dev:
        model = tiny_model[0]
        lin = Int8Linear(model, dev.put(w), dev.put(sw), n, k, ldw=ldw)
        ws = lin.workspace_bytes(m)
        scratch = (dev.raw(ws), ws)
        o1, o2, o3, q, s = dev.raw(4 * m * n), dev.raw(4 * m * n), dev.raw(4 * m * n), dev.raw(m * k), dev.raw(4 * m)
        x = dev.put(bf16_bits(xs))
        lin(x, m, o1, out_dtype="f32", workspace=scratch)
        quantize_rows(model, x, m, k, q, s)
        lin.matmul(q, s, m, o2, out_dtype="f32")
        lin.matmul(dev.put(a), dev.put(sa), m, o3, out_dtype="f32")
        one, two, three = (dev.get(o, (m, n), np.float32) for o in (o1, o2, o3))
    assert np.array_equal(one, two)
    want = (a.astype(np.float64) @ w[:, :k].astype(np.float64).T) * sa.astype(np.float64)[:, None] * sw.astype(np.float64)
    assert (np.abs(three - want) <= 3.01 * F32_HALF_STEP * np.abs(want)).all()


def test_linear_rows_do_not_depend_on_their_batch(tiny_model):
    """A row's result has the same bits alone, among a few and among many rows (all kernels sum whole numbers); a row with a NaN
    or an infinity turns into NaN and leaves the others alone."""
    from q3asr import Int8Linear
    rng = np.random.default_rng(5)
    n, k = 384, 1040
    xs = _rows(rng, 700, k, "bf16")
    w, ldw, sw = _weights(rng, n, k)
    with Device() as dev:
        lin = Int8Linear(tiny_model[0], dev.put(w), dev.put(sw), n, k, ldw=ldw)

        def run(x):
            m = len(x)
            ws, o = lin.workspace_bytes(m), dev.raw(2 * m * n)
            lin(dev.put(bf16_bits(x)), m, o, workspace=(dev.raw(ws), ws))
            return dev.get(o, (m, n), np.uint16)

        full = run(xs)
        for m in (1, 2, 5, 16, 17, 40, 64, 100, 257):
            assert np.array_equal(run(xs[:m]), full[:m]), m
        for m in (3, 20, 300):
            x = xs[:m].copy()
            x[1, 5], x[2, 9] = np.nan, np.inf
            got = run(x)
            assert np.isnan(bf16_vals(got[1:3])).all()
            assert np.array_equal(np.delete(got, (1, 2), 0), np.delete(full[:m], (1, 2), 0))


def test_linear_on_two_streams_and_in_a_graph(tiny_model):
    """Two calls at once on streams of their own, and captured calls replayed with eager work in between: always the eager bits."""
    from q3asr import Int8Linear
    rng = np.random.default_rng(6)
    model = tiny_model[0]
    with Device() as dev:
        jobs = []
        for m, n, k in ((300, 512, 768), (4, 2048, 1024), (40, 256, 4096)):
            w, ldw, sw = _weights(rng, n, k)
            lin = Int8Linear(model, dev.put(w), dev.put(sw), n, k, ldw=ldw)
            ws = lin.workspace_bytes(m)
            xs = [dev.put(bf16_bits(_rows(rng, m, k, "bf16"))) for _ in range(2)]
            x, o, scratch = dev.raw(2 * m * k), dev.raw(2 * m * n), (dev.raw(ws), ws)
            want = []
            for src in xs:
                lin(src, m, o, workspace=scratch)
                want.append(dev.get(o, (m, n), np.uint16))
            jobs.append((lin, m, n, k, xs, x, o, scratch, want))
        streams = [dev.stream() for _ in jobs]
        for _ in range(3):
            for (lin, m, n, k, xs, x, o, scratch, want), s in zip(jobs, streams):
                dev.put(np.zeros((m, n), np.uint16), o)
            for (lin, m, n, k, xs, x, o, scratch, want), s in zip(jobs, streams):
                lin(xs[1], m, o, workspace=scratch, stream=s)
            for (lin, m, n, k, xs, x, o, scratch, want), s in zip(jobs, streams):
                dev.wait(s)
                assert np.array_equal(dev.get(o, (m, n), np.uint16), want[1])
        s = streams[0]
        graph = dev.capture(s, lambda: [lin(x, m, o, workspace=scratch, stream=s) for lin, m, n, k, xs, x, o, scratch, want in jobs])
        for rep in range(4):
            for lin, m, n, k, xs, x, o, scratch, want in jobs:
                dev.put(dev.get(xs[rep % 2], (m, k), np.uint16), x)
                dev.put(np.zeros((m, n), np.uint16), o)
            assert dev.h.hipGraphLaunch(graph, s) == 0
            dev.wait(s)
            for lin, m, n, k, xs, x, o, scratch, want in jobs:
                assert np.array_equal(dev.get(o, (m, n), np.uint16), want[rep % 2]), rep
                lin(xs[0], m, o, workspace=scratch)      # eager work between the replays
        dev.h.hipGraphExecDestroy(graph)
