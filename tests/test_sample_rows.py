"""Draws from rows of logits with given random numbers (fc_sample_rows_dev) against the definition in 64 bits."""
import ctypes as C

import numpy as np
import pytest

import ferrum_cpu_b200 as fcb
from ferrum_cpu_b200 import _lib, engine

torch = pytest.importorskip("torch")


def plain_draw(row, t, k, top_p, min_p, u):
    """(token, prob, how near u times the whole is to a border of the running mass, relative to the whole)"""
    row = np.where(np.isnan(row), -np.inf, row.astype(np.float64))
    best = row.max()
    if best == -np.inf:
        return -1, 0.0, 1.0
    if not t > 0:
        return int(np.argmax(row)), 1.0, 1.0
    with np.errstate(invalid="ignore"):
        w = np.where(row == best, 1.0, np.exp((row - best) / max(np.float64(np.float32(t)), 0.01)))
    stay = w >= 2.0 ** -40
    falling = np.sort(row)[::-1]
    if 0 < k < len(row):
        stay &= row >= falling[k - 1]
    if top_p < 1:
        order = np.argsort(-row, kind="stable")
        reached = np.nonzero(np.cumsum(w[order]) >= np.float64(np.float32(top_p)) * w.sum())[0]
        if len(reached):
            stay &= row >= falling[reached[0]]
    if min_p > 0:
        stay &= w >= min(np.float64(np.float32(min_p)), 1.0)
    ids = np.nonzero(stay)[0]
    cum = np.cumsum(w[ids])
    r = np.float64(np.float32(u)) * cum[-1]
    at = min(int(np.searchsorted(cum, r)), len(ids) - 1)
    return int(ids[at]), w[ids[at]] / cum[-1], float(np.abs(cum - r).min() / cum[-1])


def draw(logits, params, u, ld=None, with_prob=True, stream=None):
    n, V = logits.shape
    ld = ld or V
    buf = torch.full((n, ld), 1e30, device="cuda")
    buf[:, :V] = torch.as_tensor(logits)
    p = np.zeros(n, dtype=[("t", "f4"), ("k", "i4"), ("p", "f4"), ("m", "f4")])
    for i, x in enumerate(params):
        p[i] = tuple(x)
    pd, ud = torch.from_numpy(p.view(np.float32).reshape(n, 4).copy()).cuda(), torch.as_tensor(np.asarray(u, np.float32)).cuda()
    token, prob = torch.full((n,), -9, dtype=torch.int32, device="cuda"), torch.full((n,), -9.0, device="cuda")
    engine.sample_rows_dev(buf.data_ptr(), ld, n, V, pd.data_ptr(), ud.data_ptr(), token.data_ptr(), prob.data_ptr() if with_prob else None, stream=stream)
    torch.cuda.synchronize()
    return token.cpu().numpy(), prob.cpu().numpy()


def check(logits, params, u, token, prob):
    for i, row in enumerate(logits):
        want, p, near = plain_draw(row, *params[i], u[i])
        if near > 1e-9:           # sums of up to 2^18 weights in 64 bits or fixed point differ by less
            assert token[i] == want, (i, params[i], u[i])
            assert abs(prob[i] - p) <= 2.0 ** -23 * p + 1e-12, i
        else:
            assert token[i] >= 0


def test_refusals_before_any_device():
    L, p = _lib.lib(), C.c_void_p(16)
    f = L.fc_sample_rows_dev
    assert f(0, None, 8, 1, 8, p, p, p, p, None) == _lib.FC_E_ARG and f(0, p, 8, 1, 8, p, None, p, p, None) == _lib.FC_E_ARG
    assert f(0, p, 7, 1, 8, p, p, p, p, None) == _lib.FC_E_SHAPE and f(0, p, 8, -1, 8, p, p, p, p, None) == _lib.FC_E_SHAPE
    assert f(0, p, 8, 1, 0, p, p, p, p, None) == _lib.FC_E_SHAPE and f(0, p, 1 << 25, 1, (1 << 24) + 1, p, p, p, p, None) == _lib.FC_E_SHAPE
    assert f(0, p, 8, 1, 8, C.c_void_p(20), p, p, p, None) == _lib.FC_E_ARG
    assert f(0, p, 8, 0, 8, p, p, p, p, None) == _lib.FC_OK


@pytest.mark.skipif(torch.cuda.is_available(), reason="there is a GPU")
def test_no_cpu_form():
    p = C.c_void_p(16)
    assert _lib.lib().fc_sample_rows_dev(0, p, 8, 1, 8, p, p, p, p, None) == _lib.FC_E_CUDA


FILTERS = [(1.0, 0, 1.0, 0.0), (0.8, 40, 0.95, 0.05), (1.3, 0, 0.9, 0.0), (0.7, 5, 1.0, 0.0), (1.0, 0, 1.0, 0.1), (1.5, 1000, 0.99, 0.001), (0.0, 3, 0.5, 0.5),
           (-1.0, 0, 1.0, 0.0), (0.003, 0, 1.0, 0.0), (50.0, 0, 1.0, 0.0), (50.0, 0, 0.5, 0.0), (1.0, 1, 1.0, 0.0), (1.0, 0, 0.0, 0.0), (1.0, 0, 1.0, 2.0),
           (float("nan"), 0, 1.0, 0.0), (1.0, 0, float("nan"), float("nan")), (1.0, 1 << 30, 2.0, -1.0), (1.0, -4, 0.3, 0.0)]


@pytest.mark.gpu
@pytest.mark.parametrize("V", [1, 2, 31, 100, 1023, 1024, 4097, 32000, 50257, 131072, 150001])
def test_draws_match_the_definition(V):
    rng = np.random.default_rng(V)
    n = 2 * len(FILTERS)
    logits = (2.5 * rng.standard_normal((n, V))).astype(np.float32)
    logits[len(FILTERS):] += (rng.random((len(FILTERS), V)) < 20 / V) * 6
    logits[rng.random((n, V)) < 0.05] = -np.inf
    logits[:, V // 2] = 1.0
    u = rng.random(n).astype(np.float32)
    params = FILTERS * 2
    token, prob = draw(logits, params, u, ld=V + 3)
    check(logits, params, u, token, prob)
    again, _ = draw(logits, params, u)                  # another distance of the rows
    assert np.array_equal(token, again)
    bare, untouched = draw(logits, params, u, with_prob=False)
    assert np.array_equal(token, bare) and (untouched == -9.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("V", [300, 70000])
def test_rows_with_nothing_or_little_to_draw(V):
    rows = np.full((9, V), -np.inf, np.float32)
    rows[1] = np.nan
    rows[2, 7] = -3.0                       # one id
    rows[3] = 0.0                           # all the same
    rows[4, [5, V - 2]] = np.inf            # infinities tie
    rows[5] = np.nan
    rows[5, V - 1] = -1e30
    rows[6, :] = -60.0                      # all but one under 2^-40
    rows[6, 11] = 0.0
    rows[7, [1, 2]] = [3e38, -3e38]
    rows[8] = np.linspace(0, 1, V)
    u = np.float32([0.5, 0.5, 0.9, 0.5, 0.75, 0.0, 1 - 2.0 ** -24, 0.999, 0.0])
    params = [(1.0, 0, 1.0, 0.0)] * 9
    token, prob = draw(rows, params, u)
    assert token[0] == token[1] == -1 and (prob[:2] == 0).all()
    assert token.tolist()[2:8] == [7, plain_draw(rows[3], *params[3], 0.5)[0], V - 2, V - 1, 11, 1] and token[8] == 0
    assert prob[4] == 0.5 and prob[2] == prob[5] == prob[7] == 1.0
    greedy, _ = draw(rows, [(0.0, 0, 1.0, 0.0)] * 9, u)
    assert greedy.tolist() == [-1, -1, 7, 0, 5, V - 1, 11, 1, V - 1]


@pytest.mark.gpu
@pytest.mark.parametrize("V", [64, 40000])
def test_ties_at_a_cut_all_stay(V):
    row = np.full(V, -2.0, np.float32)
    row[[3, 9, 20, 40]] = 1.0
    row[[10, 50]] = 2.0
    u = (np.arange(60) + 0.5).astype(np.float32) / 60
    # top-k 3 cuts among the four; so does a top-p that the two largest and a part of the four reach
    w = np.exp(row.astype(np.float64) - 2)
    for params in ((1.0, 3, 1.0, 0.0), (1.0, 0, (2 + 1.5 * np.exp(-1.0)) / w.sum(), 0.0), (1.0, 0, 1.0, 0.3)):
        token, prob = draw(np.tile(row, (60, 1)), [params] * 60, u)
        assert set(token) == {3, 9, 10, 20, 40, 50} and (np.diff(token) >= 0).all()
        whole = 2 + 4 * np.exp(-1.0)
        assert np.abs(prob - np.where(np.isin(token, [10, 50]), 1, np.exp(-1.0)) / whole).max() <= 2.0 ** -23


@pytest.mark.gpu
@pytest.mark.parametrize("V,n", [(9000, 3), (70000, 2), (70000, 300), (300001, 1), (1 << 20, 1), (1 << 20, 5)])
def test_cuts_among_more_ties_than_are_listed(V, n):
    """Logits in few steps: thousands of ids share the value at which a cut falls. And rows up to the longest."""
    rng = np.random.default_rng(V + n)
    rows = (np.round(2.0 * rng.standard_normal((min(n, 4), V))) / 2).astype(np.float32)
    rows = rows[np.arange(n) % len(rows)]
    u = rng.random(n).astype(np.float32)
    for params in ((1.0, 0, 0.9, 0.0), (0.7, 2000, 1.0, 0.0), (1.2, V // 2, 0.5, 0.0), (1.0, 0, 1.0, 0.01), (1.0, 0, 1 - 2.0 ** -20, 0.0)):
        token, prob = draw(rows, [params] * n, u)
        for i in range(min(n, 5)):
            want, p, near = plain_draw(rows[i], *params, u[i])
            assert near <= 1e-9 or (token[i] == want and abs(prob[i] - p) <= 2.0 ** -23 * p + 1e-12), (params, i)
    same = np.zeros((n, V), np.float32)
    token, prob = draw(same, [(1.0, 5, 0.5, 0.0)] * n, u)            # all tie: all stay
    assert (np.abs(prob - 1 / V) <= 2.0 ** -23 / V).all() and all(token[i] == plain_draw(same[i], 1.0, 5, 0.5, 0.0, u[i])[0] for i in range(min(n, 3)))


@pytest.mark.gpu
@pytest.mark.parametrize("V,near,width,far", [(300, 299, 1e-3, -10.0), (2000, 500, 1e-3, -20.0), (5000, 1000, 1e-3, -20.0), (700000, 700000, 1.0, 0.0)])
@pytest.mark.parametrize("top_p", [0.0, -1.0, 1e-30, 0.001])
def test_a_top_p_of_next_to_nothing_leaves_the_largest(V, near, width, far, top_p):
    """Hundreds of ids within a bucket of the largest: the cut is among them, and never above the largest."""
    row = np.full(V, far, np.float32)
    row[np.random.default_rng(V).permutation(V)[:near]] = np.linspace(0, width, near, dtype=np.float32)
    rows, u = np.tile(row, (3, 1)), np.float32([0.0, 0.5, 1 - 2.0 ** -24])
    for k in (0, 3, V // 2):
        params = [(1.0, k, top_p, 0.0)] * 3
        check(rows, params, u, *draw(rows, params, u))


@pytest.mark.gpu
@pytest.mark.parametrize("V", [6, 2000, 131072])
@pytest.mark.parametrize("size", [1e6, 1e9, 1e15, 1e16, 1e17, 1e18, 1e20, 1e24, 1e30, 1e38])
def test_rows_of_any_size_weigh_by_differences(V, size):
    """Ties of the largest, its neighbours, and logits a temperature or two below, at large values of either sign."""
    rng = np.random.default_rng(V)
    rows, params = [], []
    for t in (1.0, 0.7, 0.01, 50.0):
        for sign in (1, -1):
            top = np.float32(sign * size * 1.37)
            tied = np.full(V, top, np.float32)
            steps = np.full(V, top, np.float32)
            steps[rng.random(V) < 0.7] = np.nextafter(top, np.float32(-np.inf))
            steps[V // 3] = np.nextafter(np.nextafter(top, np.float32(-np.inf)), np.float32(-np.inf))
            below = (np.float64(top) - 3 * t * rng.random(V)).astype(np.float32)
            far = np.full(V, -np.inf, np.float32)
            far[[0, V - 1]] = top
            for row in (tied, steps, below, far):
                for k, p, m in ((0, 1.0, 0.0), (0, 0.6, 0.0), (2, 1.0, 0.0), (0, 1.0, 0.3)):
                    rows.append(row)
                    params.append((t, k, p, m))
    rows, u = np.stack(rows), rng.random(len(rows)).astype(np.float32)
    check(rows, params, u, *draw(rows, params, u))


@pytest.mark.gpu
@pytest.mark.parametrize("V", [7, 3000, 80000])
@pytest.mark.parametrize("forbidden", [-np.inf, np.nan])
def test_rows_masked_with_the_lowest_value_are_drawn(V, forbidden):
    """Every id that is left has the type's lowest value, or one next to it: finite, so that one of them is drawn."""
    lowest, temps = np.finfo(np.float32).min, (1.0, 0.01, 1e29, 1e30)
    rng = np.random.default_rng(V)
    rows = np.full((5, V), lowest, np.float32)
    rows[1, rng.random(V) < 0.5] = forbidden
    rows[1, 3] = lowest
    rows[2, :] = forbidden
    rows[2, V - 1] = lowest
    rows[3, V // 2] = np.nextafter(lowest, np.float32(0))
    rows[4] = np.where(rng.random(V) < 0.5, lowest, np.float32(-3.4e38))
    u = rng.random(5).astype(np.float32)
    for t in temps:
        for k, p, m in ((0, 1.0, 0.0), (2, 1.0, 0.0), (0, 0.5, 0.0), (0, 0.0, 0.0), (0, 1.0, 0.5), (3, 0.9, 0.1)):
            params = [(t, k, p, m)] * 5
            check(rows, params, u, *draw(rows, params, u))


@pytest.mark.gpu
@pytest.mark.parametrize("V", [50, 1000, 131072])
def test_every_id_is_drawn_as_often_as_its_weight_says(V):
    """u at the middle of each of 4096 even steps: an id's count is 4096 times its probability, to a step at either end."""
    rng = np.random.default_rng(1)
    row = (1.5 * rng.standard_normal(V)).astype(np.float32)
    n = 4096
    u = ((np.arange(n) + 0.5) / n).astype(np.float32)
    tokens = np.concatenate([draw(np.tile(row, (256, 1)), [(1.0, 0, 1.0, 0.0)] * 256, u[i:i + 256])[0] for i in range(0, n, 256)])
    assert (np.diff(tokens) >= 0).all()
    p = np.exp(row.astype(np.float64) - row.max())
    p /= p.sum()
    assert np.abs(np.bincount(tokens, minlength=V) - n * p).max() < 1.001


@pytest.mark.gpu
def test_captured_draws_take_new_logits_and_numbers():
    V, n = 9000, 3
    rng = np.random.default_rng(4)
    logits, u = torch.zeros((n, V), device="cuda"), torch.zeros(n, device="cuda")
    p = np.zeros((n, 4), np.float32)
    p[:, 0], p[:, 2] = 1.0, 0.9
    params, token = torch.from_numpy(p).cuda(), torch.zeros(n, dtype=torch.int32, device="cuda")
    st, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        engine.sample_rows_dev(logits.data_ptr(), V, n, V, params.data_ptr(), u.data_ptr(), token.data_ptr(),
                               stream=C.c_void_p(torch.cuda.current_stream().cuda_stream))
    for _ in range(3):
        x, r = rng.standard_normal((n, V)).astype(np.float32), rng.random(n).astype(np.float32)
        logits.copy_(torch.from_numpy(x))
        u.copy_(torch.from_numpy(r))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for i in range(n):
            want, _, near = plain_draw(x[i], 1.0, 0, 0.9, 0.0, r[i])
            assert token[i] == want or near < 1e-9


@pytest.mark.gpu
@pytest.mark.parametrize("n", [149, 256, 257, 700])
def test_every_row_of_a_mixed_batch_is_answered(n):
    """Batches whose rows differ in what they take (the largest, a plain draw, filters) come back in the order of the call."""
    rng = np.random.default_rng(n)
    logits = (rng.standard_normal((n, 500)) * 3).astype(np.float32)
    kinds = [(0.0, 0, 1.0, 0.0), (float("nan"), 5, 0.5, 0.0), (1.0, 0, 1.0, 0.0), (0.7, 20, 1.0, 0.0), (1.2, 0, 0.9, 0.1), (0.9, 499, 0.95, 0.0), (1.0, 500, 1.0, 0.0)]
    params = [kinds[i] for i in rng.integers(0, len(kinds), n)]
    u = rng.random(n).astype(np.float32)
    token, prob = draw(logits, params, u)
    greedy = [i for i in range(n) if not params[i][0] > 0]
    assert (token[greedy] == logits[greedy].argmax(1)).all() and (prob[greedy] == 1).all()
    rest = [i for i in range(n) if params[i][0] > 0]
    check(logits[rest], [params[i] for i in rest], u[rest], token[rest], prob[rest])


@pytest.mark.gpu
def test_an_unknown_device_is_refused():
    z = torch.zeros(64, device="cuda")
    with pytest.raises(fcb.FerrumCudaError) as e:
        engine.sample_rows_dev(z.data_ptr(), 8, 1, 8, z.data_ptr(), z.data_ptr(), z.data_ptr(), device=99)
    assert e.value.code == _lib.FC_E_ARG
