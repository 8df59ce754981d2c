"""The key / value cache of 4-bit levels (fc_kv4_*): what it holds, attention over it, and eviction from it, against plain forms in
64 bits."""
import ctypes as C
import math

import numpy as np
import pytest

import ferrum_cpu_b200 as fcb
from ferrum_cpu_b200 import _lib, kv4

torch = pytest.importorskip("torch")

EPS = 2.0 ** -24        # half a step of f32


# ---- the definitions, in 64 bits ------------------------------------------------------------------------
def stands_for(x):
    """What the cache holds of x [..][dim]."""
    x = np.asarray(x, np.float32).astype(np.float64)
    b = np.where(np.isnan(x), 0.0, x).reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    hi, lo = b.max(-1), b.min(-1)
    with np.errstate(over="ignore", invalid="ignore", divide="ignore"):
        d = np.clip(np.where(hi >= -lo, hi, lo) / -8.0, -65504.0, 65504.0).astype(np.float16).astype(np.float64)[..., None]
        q = np.clip(np.rint(b / d), -8, 7)
    return np.where(d == 0, 0.0, np.where(d == 0, 0.0, q) * d).reshape(x.shape)


def plain_attention(q, K, V, seen, scale):
    """One head: q [n][dim], K, V [len][dim]; row i sees seen[i] positions. (out, weights, bound of a score's error)"""
    out, P = np.zeros_like(q), np.zeros((len(q), len(K)))
    for i, n in enumerate(seen):
        if n > 0:
            s = K[:n] @ q[i] * scale
            p = np.exp(s - s.max())
            P[i, :n] = p / p.sum()
            out[i] = P[i, :n] @ V[:n]
    return out, P


def score_error(q, K, scale):
    """Largest error of a score in f32 arithmetic: a rounding of 2^-23 (the tensor core truncates) for every product and each of
    the sums over blocks, of levels that are up to 8 above what they stand for."""
    if not len(K):
        return 0.0
    return float((np.abs(q) @ (np.abs(K) + np.abs(K).max(-1, keepdims=True)).T).max() * abs(scale) * (q.shape[-1] + 8) * 2 * EPS)


class Run:
    """A cache and its oracle: values [seq][head][pos][dim] in 64 bits."""

    def __init__(self, n_seq, n_kv, dim, cap):
        self.cache = kv4.Kv4Cache(n_seq, n_kv, dim, cap)
        self.shape = (n_seq, n_kv, dim, cap)
        self.K = np.zeros((n_seq, n_kv, cap, dim))
        self.V = np.zeros((n_seq, n_kv, cap, dim))

    def put(self, k, v, rows, lens):
        n_seq, n_kv, dim, cap = self.shape
        at = 0
        for s, n in enumerate(rows):
            if 0 <= lens[s] <= cap - n:
                for store, x in ((self.K, k), (self.V, v)):
                    store[s, :, lens[s]:lens[s] + n] = stands_for(x[at:at + n].reshape(n, n_kv, dim)).transpose(1, 0, 2)
            at += n

    def read(self):
        n_seq, n_kv, dim, cap = self.shape
        k, v = (torch.empty((n_seq, cap, n_kv, dim), device="cuda") for _ in range(2))
        self.cache.read_dev(cap, k.data_ptr(), v.data_ptr())
        return k.cpu().numpy().transpose(0, 2, 1, 3), v.cpu().numpy().transpose(0, 2, 1, 3)


def dev(x, dtype=None):
    return torch.as_tensor(np.ascontiguousarray(x), dtype=dtype).cuda()


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def draws(rng, n, width):
    return (rng.standard_normal((n, width)) * np.exp(0.5 * rng.standard_normal((1, width)))).astype(np.float32)


def fill(run, rng, lens):
    """Positions 0 .. lens[s] of every sequence, and rows of another kind behind them."""
    n_seq, n_kv, dim, cap = run.shape
    stale = draws(rng, n_seq * cap, n_kv * dim) * 50
    kt, vt, zero = dev(stale), dev(-stale), ints([0] * n_seq)
    run.cache.append_dev(kt.data_ptr(), vt.data_ptr(), n_kv * dim, zero.data_ptr(), rows=[cap] * n_seq)
    run.put(stale, -stale, [cap] * n_seq, [0] * n_seq)
    if not sum(lens):
        return
    k, v = draws(rng, sum(lens), n_kv * dim), draws(rng, sum(lens), n_kv * dim)
    kd, vd = dev(k), dev(v)
    run.cache.append_dev(kd.data_ptr(), vd.data_ptr(), n_kv * dim, zero.data_ptr(), rows=lens)
    run.put(k, v, lens, [0] * n_seq)
    torch.cuda.synchronize()


def attend(run, rng, heads, lens, rows, with_new=True, mass=None, scale=0.0, pad=8, stream=None, q=None):
    """A call on rows that lie in one fused q | k | v buffer; checks what it may not touch. Returns (out, q, mass)."""
    n_seq, n_kv, dim, cap = run.shape
    total, width = sum(rows), (heads + 2 * n_kv) * dim + pad
    x = draws(rng, max(total, 1), width)
    if q is not None:
        x[:, :heads * dim] = q
    xd, lt = dev(x), ints(lens)
    out = torch.full((max(total, 1), heads * dim + 4), 7.0, device="cuda")
    k = xd.data_ptr() + 4 * heads * dim
    new = dict(k_ptr=k, v_ptr=k + 4 * n_kv * dim, ldkv=width) if with_new else {}
    mt = None if mass is None else dev(mass, torch.float32)
    run.cache.attend_dev(xd.data_ptr(), width, heads, lt.data_ptr(), out.data_ptr(), heads * dim + 4, rows=rows, scale=scale,
                         mass_ptr=None if mt is None else mt.data_ptr(), stream=stream, **new)
    if with_new:
        run.put(x[:, heads * dim:(heads + n_kv) * dim], x[:, (heads + n_kv) * dim:(heads + 2 * n_kv) * dim], rows, lens)
    torch.cuda.synchronize()
    got = out.cpu().numpy()
    assert (got[:, heads * dim:] == 7.0).all() and (lt.cpu().numpy() == lens).all()
    return got[:total, :heads * dim], x[:total, :heads * dim], None if mt is None else mt.cpu().numpy()


def check_attention(run, heads, lens, rows, got, q, with_new=True, mass=None, got_mass=None, scale=None):
    n_seq, n_kv, dim, cap = run.shape
    group, scale = heads // n_kv, scale or 1.0 / math.sqrt(dim)
    at = 0
    for s, n in enumerate(rows):
        length = lens[s] + n if with_new else lens[s]
        seen = [max(0, length - n + i + 1) for i in range(n)]
        for h in range(n_kv):
            K, V = run.K[s, h, :length], run.V[s, h, :length]
            received = np.zeros(length)
            slack = 0.0
            for g in range(group):
                c = (h * group + g) * dim
                qq = q[at:at + n, c:c + dim].astype(np.float64)
                want, P = plain_attention(qq, K, V, seen, scale)
                ds = score_error(qq, K, scale) if n else 0.0
                top = np.abs(V).max() if length else 0.0
                # weights: twice a score's error, 2^-20 for the exponential and two f16 planes; sums: a rounding for each tile of 64 positions
                tol = top * (2 * ds + 2.0 ** -20 + (length / 64 + 64) * 2 * EPS)
                assert np.abs(got[at:at + n, c:c + dim] - want).max(initial=0.0) <= tol, (s, h, g, n, length)
                received += P.sum(0)
                slack = max(slack, 2 * ds)
            if mass is not None:
                old = lens[s] if with_new else length
                want = np.where(np.arange(length) < old, mass[s, h, :length], 0.0) + received
                m = got_mass[s, h]
                assert (np.abs(m[:length] - want) <= want * (slack + 2.0 ** -20 + (n * group + 8) * EPS) + 1e-30).all(), (s, h)
                assert (m[length:] == mass[s, h, length:].astype(np.float32)).all()
        at += n


# ---- refusals, before any device is used ------------------------------------------------------------------
def test_create_refuses_what_it_does_not_cover():
    for args, code in (((0, 1, 64, 8), _lib.FC_E_SHAPE), ((257, 1, 64, 8), _lib.FC_E_SHAPE), ((1, 0, 64, 8), _lib.FC_E_SHAPE), ((1, 1, 48, 8), _lib.FC_E_SHAPE),
                       ((1, 1, 288, 8), _lib.FC_E_SHAPE), ((1, 1, 0, 8), _lib.FC_E_SHAPE), ((1, 1, 64, 0), _lib.FC_E_SHAPE), ((1, 1, 64, (1 << 24) + 1), _lib.FC_E_SHAPE)):
        with pytest.raises(fcb.FerrumCudaError) as e:
            kv4.Kv4Cache(*args)
        assert e.value.code == code


def test_null_handles_are_refused():
    L = _lib.lib()
    one = C.c_void_p(16)
    assert L.fc_kv4_append_dev(None, one, one, 64, None, one, None) == _lib.FC_E_ARG
    assert L.fc_kv4_attend_dev(None, one, 64, 1, None, None, 0, None, one, 0.0, None, one, 64, None) == _lib.FC_E_ARG
    assert L.fc_kv4_read_dev(None, None, 1, one, one, None) == _lib.FC_E_ARG
    assert L.fc_kv4_evict_dev(None, None, one, one, 1, 0, one, None, None, None) == _lib.FC_E_ARG
    L.fc_kv4_free(None)


@pytest.mark.skipif(torch.cuda.is_available(), reason="there is a GPU")
def test_no_cpu_form():
    with pytest.raises(fcb.FerrumCudaError) as e:
        kv4.Kv4Cache(1, 1, 64, 8)
    assert e.value.code == _lib.FC_E_CUDA


@pytest.mark.gpu
def test_calls_refuse_what_does_not_fit():
    c = kv4.Kv4Cache(2, 2, 64, 8)
    p = torch.zeros(4096, device="cuda").data_ptr()
    lens = ints([0, 0])
    lp = lens.data_ptr()

    def code(f, *a, **k):
        with pytest.raises(fcb.FerrumCudaError) as e:
            f(*a, **k)
        return e.value.code
    assert code(c.append_dev, p, None, 128, lp) == _lib.FC_E_ARG
    assert code(c.append_dev, p + 4, p, 128, lp) == _lib.FC_E_ARG
    assert code(c.append_dev, p, p, 126, lp) == _lib.FC_E_SHAPE and code(c.append_dev, p, p, 124, lp) == _lib.FC_E_SHAPE
    assert code(c.append_dev, p, p, 128, lp, rows=[9, 0]) == _lib.FC_E_DIM
    assert code(c.append_dev, p, p, 128, lp, rows=[-1, 0]) == _lib.FC_E_SHAPE
    assert code(c.append_dev, p, p, 128, lp, rows=[1]) == _lib.FC_E_SHAPE
    a = c.attend_dev
    assert code(a, p, 256, 3, lp, p, 256) == _lib.FC_E_DIM and code(a, p, 256, 0, lp, p, 256) == _lib.FC_E_DIM
    assert code(a, p, 252, 4, lp, p, 256) == _lib.FC_E_SHAPE and code(a, p, 256, 4, lp, p, 258) == _lib.FC_E_SHAPE
    assert code(a, p, 256, 4, lp, p, 256, k_ptr=p) == _lib.FC_E_ARG and code(a, p, 256, 4, lp, p, 256, scale=math.inf) == _lib.FC_E_ARG
    assert code(a, p, 256, 4, lp, p, 256, k_ptr=p, v_ptr=p, ldkv=64) == _lib.FC_E_SHAPE
    assert code(a, p + 8, 256, 4, lp, p, 256) == _lib.FC_E_ARG and code(a, p, 256, 4, None, p, 256) == _lib.FC_E_ARG
    assert code(c.read_dev, -1, p, p) == _lib.FC_E_SHAPE and code(c.read_dev, 1, p, None) == _lib.FC_E_ARG
    d, other = kv4.Kv4Cache(2, 2, 64, 4), kv4.Kv4Cache(2, 1, 64, 4)
    m = torch.zeros((2, 2, 8), device="cuda").data_ptr()
    lo = ints([0, 0]).data_ptr()
    assert code(c.evict_dev, c, lp, lo, 4, 0, m) == _lib.FC_E_ARG and code(c.evict_dev, d, lp, lp, 4, 0, m) == _lib.FC_E_ARG
    assert code(c.evict_dev, other, lp, lo, 4, 0, m) == _lib.FC_E_DIM and code(c.evict_dev, d, lp, lo, 5, 0, m) == _lib.FC_E_DIM
    assert code(c.evict_dev, d, lp, lo, 0, 0, m) == _lib.FC_E_SHAPE and code(c.evict_dev, d, lp, lo, 4, 5, m) == _lib.FC_E_SHAPE
    assert code(c.evict_dev, d, lp, lo, 4, 0, None) == _lib.FC_E_ARG
    c.attend_dev(p, 256, 4, lp, p, 256, rows=[0, 0])         # nothing to do
    c.read_dev(0, p, p)
    torch.cuda.synchronize()


# ---- what the cache holds -----------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 160, 192, 224, 256])
def test_append_and_read_hold_the_definition_to_the_bit(dim):
    rng = np.random.default_rng(dim)
    run = Run(3, 2, dim, 70)
    lens, rows = [0, 13, 64], [70, 5, 0]
    k, v = draws(rng, 75, 2 * dim), draws(rng, 75, 2 * dim)
    k[0, :32] = 0.0                                                  # a block of zeros
    k[1, :32] = np.linspace(-8, 7.75, 32)                            # ties between levels, and of magnitude below
    k[2, :32] = np.tile([1.0, -1.0], 16)
    k[3, :32] = 1e-9                                                 # the scale is no f16
    k[4, :32] = np.linspace(-3e-6, 3e-6, 32)                         # a subnormal scale
    v[5, :32] = 3e38
    v[6, :3] = [np.inf, -np.inf, np.nan]
    v[7, :32] = np.nan
    v[8, :32] = -0.0
    v[9, :4] = [1e6, -1e6, 524288.0, 65504.0]
    kd, vd, lt = dev(k), dev(v), ints(lens)
    run.cache.append_dev(kd.data_ptr(), vd.data_ptr(), 2 * dim, lt.data_ptr(), rows=rows)
    run.put(k, v, rows, lens)
    gk, gv = run.read()
    assert np.array_equal(gk, run.K.astype(np.float32)) and np.array_equal(gv, run.V.astype(np.float32))


@pytest.mark.gpu
def test_read_begins_where_each_sequence_says():
    rng = np.random.default_rng(2)
    run = Run(3, 1, 64, 9)
    fill(run, rng, [9, 4, 7])
    k, v = (torch.empty((3, 4, 1, 64), device="cuda") for _ in range(2))
    start = ints([-2, 3, 8])
    run.cache.read_dev(4, k.data_ptr(), v.data_ptr(), from_ptr=start.data_ptr())
    for s, at in enumerate([-2, 3, 8]):
        for i in range(4):
            inside = 0 <= at + i < 9
            for got, held in ((k, run.K), (v, run.V)):
                assert np.array_equal(got[s, i, 0].cpu().numpy(), held[s, 0, at + i].astype(np.float32) if inside else np.zeros(64, np.float32))


# ---- attention -------------------------------------------------------------------------------------------------
CASES = [  # heads, kv, dim, cached, rows
    (1, 1, 32, [0], [1]),
    (8, 2, 64, [33], [1]),
    (4, 4, 64, [0, 1, 63, 64, 65], [1] * 5),
    (14, 2, 64, [127, 500, 3], [1, 0, 2]),
    (12, 1, 96, [300, 17], [1, 1]),
    (32, 8, 64, [1023], [1]),
    (8, 8, 128, [1000, 0, 200], [5, 4, 1]),
    (16, 2, 128, [640, 31], [3, 7]),
    (3, 1, 160, [70], [9]),
    (2, 2, 192, [65, 5], [2, 70]),
    (6, 2, 224, [129], [1]),
    (8, 1, 256, [400, 40], [1, 33]),
    (4, 2, 64, [0], [130]),
    (8, 2, 32, [100, 0, 7], [64, 129, 1]),
    (6, 2, 96, [0, 250], [200, 65]),
    (4, 4, 128, [1, 77], [191, 66]),
    (20, 1, 64, [45], [40]),
    (64, 1, 64, [260, 2], [1, 1]),
    (2, 1, 256, [0], [150]),
]


@pytest.mark.gpu
@pytest.mark.parametrize("with_mass", [False, True])
@pytest.mark.parametrize("heads,kv,dim,lens,rows", CASES)
def test_attention_over_cached_and_new_rows(heads, kv, dim, lens, rows, with_mass):
    rng = np.random.default_rng(heads * 1000 + dim + sum(rows))
    cap = max(a + b for a, b in zip(lens, rows)) + 3
    run = Run(len(lens), kv, dim, cap)
    fill(run, rng, lens)
    mass = rng.random((len(lens), kv, cap)).astype(np.float32) if with_mass else None
    got, q, m = attend(run, rng, heads, lens, rows, mass=mass)
    check_attention(run, heads, lens, rows, got, q, mass=mass, got_mass=m)
    gk, gv = run.read()
    assert np.array_equal(gk, run.K.astype(np.float32)) and np.array_equal(gv, run.V.astype(np.float32))


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,dim,lens,rows", [(8, 2, 64, [33, 1, 0], [1, 1, 1]), (6, 3, 128, [200, 70, 3], [66, 1, 5]), (4, 1, 32, [513], [1])])
def test_attention_over_what_is_cached(heads, kv, dim, lens, rows):
    """Without new rows the queries are the last positions; a row before the first position sees nothing and is zeros."""
    rng = np.random.default_rng(dim)
    run = Run(len(lens), kv, dim, max(lens) + 1)
    fill(run, rng, lens)
    mass = rng.random((len(lens), kv, max(lens) + 1)).astype(np.float32)
    before = run.read()
    got, q, m = attend(run, rng, heads, lens, rows, with_new=False, mass=mass, scale=0.25)
    check_attention(run, heads, lens, rows, got, q, with_new=False, mass=mass, got_mass=m, scale=0.25)
    assert all(np.array_equal(a, b) for a, b in zip(before, run.read()))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [[1, 1, 1, 1, 1], [3, 3, 2, 3, 100]])
def test_sequences_whose_length_is_none(rows):
    """Negative, or no room for the rows: their rows are NaN, nothing of theirs changes, the others are as ever."""
    rng = np.random.default_rng(3)
    run = Run(5, 2, 64, 130)
    good = [40, 40, 129 - rows[2], 0, 30]
    fill(run, rng, good)
    mass = rng.random((5, 2, 130)).astype(np.float32)
    lens = [-1, 131 - rows[1], 130 - rows[2], 0, 1 << 30]
    kept = run.read()
    got, q, m = attend(run, rng, 4, lens, rows, mass=mass)
    at = np.cumsum([0] + rows)
    for s in (0, 1, 4):
        assert np.isnan(got[at[s]:at[s + 1]]).all() and np.array_equal(m[s], mass[s])
    gk, gv = run.read()
    for s in (0, 1, 4):
        assert np.array_equal(gk[s], kept[0][s]) and np.array_equal(gv[s], kept[1][s])
    live = [0 if s in (0, 1, 4) else n for s, n in enumerate(rows)]
    part = np.concatenate([np.arange(at[s], at[s + 1]) for s in (2, 3)])
    check_attention(run, 4, [0, 0, lens[2], 0, 0], live, got[part], q[part], mass=np.where(np.array([0, 0, 1, 1, 0])[:, None, None] == 1, mass, m), got_mass=m)
    nan, _, _ = attend(run, rng, 4, [131, 10, 10, 10, 10], [1] * 5, with_new=False)
    assert np.isnan(nan[0]).all() and np.isfinite(nan[1:]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 90])
def test_what_lies_behind_a_row_does_not_reach_it(rows):
    """Behind the last position: rows as large as the cache holds. Among the call's own rows: a later one of infinities."""
    outs = []
    for stale in (0.0, 3e38):
        rng = np.random.default_rng(5)
        run = Run(1, 2, 64, 300)
        s = np.full((300, 128), stale, np.float32)
        sd, zero = dev(s), ints([0])
        run.cache.append_dev(sd.data_ptr(), sd.data_ptr(), 128, zero.data_ptr(), rows=[300])
        k, lt = dev(draws(rng, 150, 128)), ints([150])
        run.cache.append_dev(k.data_ptr(), k.data_ptr(), 128, zero.data_ptr(), rows=[150])
        x = draws(rng, rows, 512)
        x[rows - 1, 256:] = np.inf if stale and rows > 1 else x[rows - 1, 256:]
        xd, out = dev(x), torch.empty((rows, 256), device="cuda")
        run.cache.attend_dev(xd.data_ptr(), 512, 4, lt.data_ptr(), out.data_ptr(), 256, k_ptr=xd.data_ptr() + 1024, v_ptr=xd.data_ptr() + 1536, ldkv=512,
                             rows=[rows])
        outs.append(out.cpu().numpy())
    n = rows - 1 if rows > 1 else 1
    assert np.array_equal(outs[0][:n], outs[1][:n])


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 80])
def test_queries_of_any_size_and_none(rows):
    """NaN in one head's query stays there; queries of 1e-20 and 1e20 times the usual size: even weights, and all of it on the largest."""
    rng = np.random.default_rng(6)
    run = Run(1, 2, 64, 200)
    fill(run, rng, [100])
    q = draws(rng, rows, 6 * 64)
    q[0, 64:128] = np.nan
    q[0, 128:192] *= 1e-20
    q[0, 192:256] *= 1e20
    q[0, 256:320] = 0.0
    got, q, _ = attend(run, rng, 6, [100], [rows], q=q)
    assert np.isnan(got[0, 64:128]).all()
    ok = np.nan_to_num(q.astype(np.float64))
    for head in (0, 2, 3, 4, 5):
        h = head // 3
        want, P = plain_attention(ok[:1, head * 64:(head + 1) * 64], run.K[0, h, :101], run.V[0, h, :101], [101], 0.125)
        top = np.abs(run.V[0, h, :101]).max()
        ds = score_error(ok[:1, head * 64:(head + 1) * 64], run.K[0, h, :101], 0.125)
        if head == 3:
            s = run.K[0, h, :101] @ ok[0, 192:256] * 0.125
            assert np.sort(s)[-1] - np.sort(s)[-2] > 4 * ds + 100      # one position has all of the weight, whatever the rounding
            ds = 0.0
        assert np.abs(got[0, head * 64:(head + 1) * 64] - want[0]).max() <= top * (2 * ds + 2.0 ** -20 + 66 * 2 * EPS)
    if rows > 1:
        assert np.isfinite(got[1:]).all()


@pytest.mark.gpu
def test_values_of_very_different_size_keep_their_own_precision():
    """Blocks of a head whose values lie 2^12 apart, and values as small as 2^-18: each to its own size."""
    rng = np.random.default_rng(8)
    n, dim = 257, 128
    run = Run(1, 1, dim, n + 40)
    k, v = draws(rng, n, dim), rng.standard_normal((n, dim)).astype(np.float32)
    v *= np.repeat(np.float32([1.0, 2.0 ** -12, 2.0 ** -6, 2.0 ** -18]), 32)
    kd, vd, zero, lt = dev(k), dev(v), ints([0]), ints([n])
    run.cache.append_dev(kd.data_ptr(), vd.data_ptr(), dim, zero.data_ptr(), rows=[n])
    run.put(k, v, [n], [0])
    for rows in (1, 33):
        q = draws(rng, rows, 4 * dim) * np.float32(0.3)
        qd, out = dev(q), torch.empty((rows, 4 * dim), device="cuda")
        run.cache.attend_dev(qd.data_ptr(), 4 * dim, 4, lt.data_ptr(), out.data_ptr(), 4 * dim, rows=[rows])
        got = out.cpu().numpy()
        for g in range(4):
            qq = q[:, g * dim:(g + 1) * dim].astype(np.float64)
            want, _ = plain_attention(qq, run.K[0, 0, :n], run.V[0, 0, :n], [n - rows + i + 1 for i in range(rows)], 1 / math.sqrt(dim))
            ds = score_error(qq, run.K[0, 0, :n], 1 / math.sqrt(dim))
            for b in range(4):
                at = slice(32 * b, 32 * b + 32)
                top = np.abs(run.V[0, 0, :n, at]).max()
                # the planes of a weight times its scale keep 2^-22 of the largest scale in a tile at 2^14: 2^-38 of it
                assert np.abs(got[:, g * dim:(g + 1) * dim][:, at] - want[:, at]).max() <= top * (2 * ds + 2.0 ** -20 + 70 * 2 * EPS) + 2.0 ** -36, b


@pytest.mark.gpu
@pytest.mark.parametrize("kv,rows", [(16384, 32), (8192, 32), (16384, 24), (65535, 3), (65535, 9)])
@pytest.mark.parametrize("with_mass", [False, True])
def test_heads_by_the_ten_thousand(kv, rows, with_mass):
    rng = np.random.default_rng(13)
    run = Run(1, kv, 32, rows + 2)
    fill(run, rng, [2])
    mass = rng.random((1, kv, rows + 2)).astype(np.float32) if with_mass else None
    got, q, m = attend(run, rng, kv, [2], [rows], mass=mass)
    some = rng.integers(0, kv, 200)                              # heads of their own: a part of them is a call of its own
    part = Run(1, len(some), 32, rows + 2)
    part.K, part.V = run.K[:, some], run.V[:, some]
    pick = lambda x: x.reshape(rows, kv, 32)[:, some].reshape(rows, -1)  # noqa: E731
    check_attention(part, len(some), [2], [rows], pick(got), pick(q), mass=mass[:, some] if with_mass else None, got_mass=m[:, some] if with_mass else None)
    assert np.isfinite(got).all()
    k, v = run.read()
    assert np.array_equal(k[0, some], run.K[0, some]) and np.array_equal(v[0, some], run.V[0, some])


@pytest.mark.gpu
def test_a_cache_that_finds_no_memory_fails_alone():
    run, rng = Run(1, 2, 64, 40), np.random.default_rng(14)
    fill(run, rng, [10])
    for _ in range(2):
        with pytest.raises(fcb.FerrumCudaError) as e:
            kv4.Kv4Cache(256, 65535, 256, 1 << 24)               # some 10^17 bytes
        assert e.value.code == _lib.FC_E_CUDA
        got, q, _ = attend(run, rng, 4, [10], [2])
        check_attention(run, 4, [10], [2], got, q)
        assert np.array_equal(run.read()[0], run.K)
        torch.zeros(8, device="cuda").add_(1)                    # nor does another library's launch


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1.0, 2.0 ** -8, 2.0 ** -14, 2.0 ** -19])
@pytest.mark.parametrize("rows,heads", [(33, 4), (33, 2), (5, 4)])
def test_values_beside_rows_of_zeros_keep_their_precision(size, rows, heads):
    """Two positions of three hold zeros: small values of the third are as exact as large ones."""
    rng = np.random.default_rng(11)
    n, dim = 35, 64
    run = Run(1, 1, dim, n)
    k, v = draws(rng, n, dim), (size * rng.standard_normal((n, dim))).astype(np.float32)
    v[np.arange(n) % 3 != 0] = 0.0
    kd, vd, zero, lt = dev(k), dev(v), ints([0]), ints([n])
    run.cache.append_dev(kd.data_ptr(), vd.data_ptr(), dim, zero.data_ptr(), rows=[n])
    run.put(k, v, [n], [0])
    q = draws(rng, rows, heads * dim) * np.float32(0.05)
    qd, out = dev(q), torch.empty((rows, heads * dim), device="cuda")
    run.cache.attend_dev(qd.data_ptr(), heads * dim, heads, lt.data_ptr(), out.data_ptr(), heads * dim, rows=[rows])
    got = out.cpu().numpy()
    for g in range(heads):
        qq = q[:, g * dim:(g + 1) * dim].astype(np.float64)
        want, _ = plain_attention(qq, run.K[0, 0, :n], run.V[0, 0, :n], [n - rows + i + 1 for i in range(rows)], 1 / math.sqrt(dim))
        ds, top = score_error(qq, run.K[0, 0, :n], 1 / math.sqrt(dim)), np.abs(run.V[0, 0, :n]).max()
        # as in check_attention; a score with a power of two of up to 2^5 added is rounded to 2^-20, which its weight takes times ln 2
        assert np.abs(got[:, g * dim:(g + 1) * dim] - want).max() <= top * (2 * ds + 2 * 2.0 ** -20 + 65 * 2 * EPS)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,dim", [(8, 2, 64), (4, 4, 128)])
def test_a_prompt_is_its_rows_one_by_one(heads, kv, dim):
    rng = np.random.default_rng(9)
    n = 75
    x = draws(rng, n, (heads + 2 * kv) * dim)
    xd, ld = dev(x), (heads + 2 * kv) * dim
    a, b = kv4.Kv4Cache(1, kv, dim, n), kv4.Kv4Cache(1, kv, dim, n)
    whole, single = torch.empty((n, heads * dim), device="cuda"), torch.empty((n, heads * dim), device="cuda")
    mass = torch.zeros((2, kv, n), device="cuda")
    lens = [ints([i]) for i in range(n)]
    k = heads * dim * 4
    a.attend_dev(xd.data_ptr(), ld, heads, lens[0].data_ptr(), whole.data_ptr(), heads * dim, k_ptr=xd.data_ptr() + k, v_ptr=xd.data_ptr() + k + 4 * kv * dim,
                 ldkv=ld, rows=[n], mass_ptr=mass[0].data_ptr())
    for i in range(n):
        row = xd[i].data_ptr()
        b.attend_dev(row, ld, heads, lens[i].data_ptr(), single[i].data_ptr(), heads * dim, k_ptr=row + k, v_ptr=row + k + 4 * kv * dim, ldkv=ld,
                     mass_ptr=mass[1].data_ptr())
    ra, rb = torch.empty((2, 1, n, kv, dim), device="cuda"), torch.empty((2, 1, n, kv, dim), device="cuda")
    a.read_dev(n, ra[0].data_ptr(), ra[1].data_ptr())
    b.read_dev(n, rb[0].data_ptr(), rb[1].data_ptr())
    assert torch.equal(ra, rb)
    q = x[:, :heads * dim].astype(np.float64).reshape(n, heads, dim)
    K = ra[0, 0].double().cpu().numpy()
    ds = max(score_error(q[:, h], K[:, h * kv // heads], 1 / math.sqrt(dim)) for h in range(heads))
    top = float(ra[1].abs().max())
    assert float((whole - single).abs().max()) <= 2 * top * (2 * ds + 2.0 ** -20 + 66 * 2 * EPS)
    assert float(((mass[0] - mass[1]).abs() - mass[0] * 2 * (2 * ds + 2.0 ** -20 + (n * heads // kv + 8) * EPS)).max()) <= 0


@pytest.mark.gpu
def test_calls_repeat_to_the_bit_and_on_streams_of_their_own():
    rng = np.random.default_rng(10)
    streams = [torch.cuda.Stream() for _ in range(3)]
    runs = [Run(2, 2, 64, 700) for _ in streams]
    x = dev(draws(rng, 2 * 320, 8 * 64))
    lens = ints([350, 0])
    outs = [[torch.empty((640, 256), device="cuda") for _ in range(4)] for _ in streams]
    masses = [torch.zeros((4, 2, 2, 700), device="cuda") for _ in streams]
    base = dev(draws(rng, 350, 2 * 64))
    zero = ints([0, 0])
    torch.cuda.synchronize()
    for i in range(4):
        for run, st, out, mass in zip(runs, streams, outs, masses):
            s = C.c_void_p(st.cuda_stream)
            run.cache.append_dev(base.data_ptr(), base.data_ptr(), 128, zero.data_ptr(), rows=[350, 0], stream=s)
            run.cache.attend_dev(x.data_ptr(), 512, 4, lens.data_ptr(), out[i].data_ptr(), 256, k_ptr=x.data_ptr() + 1024, v_ptr=x.data_ptr() + 1536, ldkv=512,
                                 rows=[320, 320], mass_ptr=mass[i].data_ptr(), stream=s)
    torch.cuda.synchronize()
    for out, mass in zip(outs, masses):
        assert all(torch.equal(out[i], outs[0][0]) and torch.equal(mass[i], masses[0][0]) for i in range(4))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [None, [1, 3], [40, 1]])
def test_a_captured_call_reads_the_lengths_anew(rows):
    rng = np.random.default_rng(11)
    run, twin = Run(2, 2, 64, 400), Run(2, 2, 64, 400)
    counts = rows or [1, 1]
    total = sum(counts)
    x, lens, out, mass = dev(draws(rng, total, 8 * 64)), ints([0, 0]), torch.empty((total, 256), device="cuda"), torch.zeros((2, 2, 400), device="cuda")

    def call(cache, st):
        cache.attend_dev(x.data_ptr(), 512, 4, lens.data_ptr(), out.data_ptr(), 256, k_ptr=x.data_ptr() + 1024, v_ptr=x.data_ptr() + 1536, ldkv=512, rows=rows,
                         mass_ptr=mass.data_ptr(), stream=C.c_void_p(st.cuda_stream))
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            call(run.cache, torch.cuda.current_stream())
    for a, b in ([0, 0], [40, 3], [41, 360], [200, 70]):
        x.copy_(dev(draws(rng, total, 8 * 64)))
        lens.copy_(ints([a, b]))
        mass.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got, m = out.clone(), mass.clone()
        mass.zero_()
        call(twin.cache, torch.cuda.current_stream())
        torch.cuda.synchronize()
        assert torch.equal(got, out) and torch.equal(m, mass)
    for a, b in zip(run.read(), twin.read()):
        assert np.array_equal(a, b)


@pytest.mark.gpu
def test_the_most_sequences_and_few_with_rows():
    rng = np.random.default_rng(13)
    run = Run(256, 1, 32, 40)
    lens = [int(v) for v in rng.integers(0, 38, 256)]
    fill(run, rng, lens)
    rows = [0] * 256
    for s in (0, 3, 77, 200, 255):
        rows[s] = 2
    got, q, _ = attend(run, rng, 3, lens, rows)
    check_attention(run, 3, lens, rows, got, q)
    got, q, _ = attend(run, rng, 2, lens, [1] * 256)
    check_attention(run, 2, lens, [1] * 256, got, q)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 3])
def test_positions_past_32_bits(rows):
    """Eight heads of 2^24 positions of 256: words and halves lie past 2^32. The rows at the end see nothing but zeros, whose scores are 0:
    the weight of a new row with score s is e^s / (2^24 - rows + sums of e^s)."""
    cap, kv, dim = 1 << 24, 8, 256
    c = kv4.Kv4Cache(1, kv, dim, cap)
    x = np.zeros((rows, 3 * kv * dim), np.float32)
    level = np.where(np.arange(dim) % 32 == 0, 1.0, 0.5).astype(np.float32)         # exact in 4 bits: 8 and 4 eighths
    x[:, :kv * dim] = 17.0 / 16 / np.tile(level, kv) / (dim / 256)                  # q k / 16 = 17
    x[:, kv * dim:2 * kv * dim] = -np.tile(level, kv)
    x[:, :kv * dim] *= -1
    x[:, 2 * kv * dim:] = -np.tile(level, kv) * np.repeat(np.arange(1, kv + 1), dim)
    xd, lens, out = dev(x), ints([cap - rows]), torch.empty((rows, kv * dim), device="cuda")
    c.attend_dev(xd.data_ptr(), 3 * kv * dim, kv, lens.data_ptr(), out.data_ptr(), kv * dim, k_ptr=xd.data_ptr() + 4 * kv * dim, v_ptr=xd.data_ptr() + 8 * kv * dim,
                 ldkv=3 * kv * dim, rows=[rows])
    got = out.cpu().numpy().astype(np.float64)
    for i in range(rows):
        w = (i + 1) * math.exp(17.0) / (cap - rows + (i + 1) * math.exp(17.0))
        want = w * x[i, 2 * kv * dim:]
        # a score of 17 in f32: 17 * 264 roundings at the most
        assert np.abs(got[i] - want).max() <= np.abs(want).max() * (17 * 264 * 2 * EPS + 2.0 ** -18)
    k, v = (torch.empty((1, 4, kv, dim), device="cuda") for _ in range(2))
    start = ints([cap - 4])
    c.read_dev(4, k.data_ptr(), v.data_ptr(), from_ptr=start.data_ptr())
    for t, at in ((k, kv * dim), (v, 2 * kv * dim)):
        assert np.array_equal(t[0, 4 - rows:].cpu().numpy().reshape(rows, -1), x[:, at:at + kv * dim]) and not t[0, :4 - rows].any()
    c.close()


# ---- eviction ------------------------------------------------------------------------------------------------------
def plain_kept(mass, length, budget, recent):
    if length <= budget:
        return list(range(length))
    old = length - recent
    key = np.where(np.isnan(mass[:old]), -np.inf, mass[:old])
    order = sorted(range(old), key=lambda j: (-key[j], np.isnan(mass[j]), j))
    return sorted(order[:budget - recent]) + list(range(old, length))


@pytest.mark.gpu
@pytest.mark.parametrize("kv,dim,lens,budget,recent", [
    (1, 64, [100], 50, 10), (2, 64, [1152, 1024, 1, 0], 1024, 256), (2, 128, [513, 700, 64], 64, 64), (1, 32, [65], 64, 0), (3, 96, [300, 299], 299, 3),
    (1, 256, [77, 3], 1, 0), (1, 160, [130], 2, 1), (2, 64, [9000, 5000], 2048, 128), (1, 64, [20000], 33, 32)])
def test_eviction_keeps_the_recent_and_the_heaviest(kv, dim, lens, budget, recent):
    rng = np.random.default_rng(budget)
    cap = max(lens) + 5
    run, to = Run(len(lens), kv, dim, cap), Run(len(lens), kv, dim, budget + 2)
    fill(run, rng, lens)
    fill(to, rng, [budget + 2] * len(lens))
    before = to.read()
    mass = rng.random((len(lens), kv, cap)).astype(np.float32) ** 6
    mass[rng.random(mass.shape) < 0.2] = 0.0
    mass[:, :, 3::7] = mass[:, :, 3:4]                          # ties, at a weight that may be the last to stay
    mass[:, :, 5:9] = np.float32([-0.0, np.nan, np.inf, -1.0])[:mass[:, :, 5:9].shape[2]]
    md, lt, left = dev(mass), ints(lens), torch.full((len(lens),), -5, dtype=torch.int32, device="cuda")
    out, kept = torch.full((len(lens), kv, budget + 2), 9.0, device="cuda"), torch.full((len(lens), kv, budget), -7, dtype=torch.int32, device="cuda")
    run.cache.evict_dev(to.cache, lt.data_ptr(), left.data_ptr(), budget, recent, md.data_ptr(), out.data_ptr(), kept.data_ptr())
    gk, gv = to.read()
    assert left.tolist() == [min(n, budget) for n in lens] and lt.tolist() == lens
    for s, n in enumerate(lens):
        for h in range(kv):
            want = plain_kept(mass[s, h], n, budget, recent)
            assert kept[s, h].tolist() == want + [-1] * (budget - len(want)), (s, h)
            m = len(want)
            assert np.array_equal(out[s, h, :m].cpu().numpy(), mass[s, h, want], equal_nan=True) and (out[s, h, m:] == 9.0).all()
            assert np.array_equal(gk[s, h, :m], run.K[s, h, want].astype(np.float32)) and np.array_equal(gv[s, h, :m], run.V[s, h, want].astype(np.float32))
            assert np.array_equal(gk[s, h, m:], before[0][s, h, m:]) and np.array_equal(gv[s, h, m:], before[1][s, h, m:])


@pytest.mark.gpu
def test_eviction_of_lengths_that_are_none():
    run, to = Run(3, 1, 64, 20), Run(3, 1, 64, 8)
    fill(run, np.random.default_rng(1), [20, 20, 20])
    mass, left = torch.rand((3, 1, 20), device="cuda"), ints([0, 0, 0])
    kept = torch.empty((3, 1, 8), dtype=torch.int32, device="cuda")
    lens = ints([-3, 500, 20])
    run.cache.evict_dev(to.cache, lens.data_ptr(), left.data_ptr(), 8, 2, mass.data_ptr(), kept_ptr=kept.data_ptr())
    # a negative length is none, one past the capacity the whole cache
    assert left.tolist() == [0, 8, 8] and kept[0].tolist() == [[-1] * 8]
    for s in (1, 2):
        assert kept[s, 0].tolist() == plain_kept(mass[s, 0].cpu().numpy(), 20, 8, 2)
