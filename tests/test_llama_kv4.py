"""The Llama decoder on a cache of 4-bit levels (fc_llama_cache_create_kv4): prompts, steps, generation and evictions against the
same decoder in 64 bits, and the serving loop of its operators together."""
import ctypes as C
import math

import numpy as np
import pytest

import ferrum_cpu_b200 as fcb
from ferrum_cpu_b200 import _lib, engine, kv4, synth
from ferrum_cpu_b200.llama import CudaLlama
from tests.test_kv4 import dev, draws, ints, plain_attention, plain_kept, score_error, stands_for
from tests.test_sample_rows import plain_draw

torch = pytest.importorskip("torch")


class Plain:
    """The decoder in 64 bits, its keys and values through stands_for; with a capacity, cut down as the cache is."""

    def __init__(self, sm, capacity=None, budget=0, recent=0):
        D = self.D = sm.dims
        mat = lambda raw, n, k: synth.q8_0_dequantize(raw, n * k).reshape(n, k).astype(np.float64)  # noqa: E731
        d, F, qd, kvd = D["d_model"], D["d_ff"], D["n_head"] * D["head_dim"], D["n_kv_head"] * D["head_dim"]
        self.tok = mat(sm.token_embd, D["vocab"], d)
        self.norm = sm.output_norm.astype(np.float64)
        self.layers = [{"wq": mat(L["wq_q8"], qd, d), "wk": mat(L["wk_q8"], kvd, d), "wv": mat(L["wv_q8"], kvd, d), "wo": mat(L["wo_q8"], d, qd),
                        "gate": mat(L["gate_q8"], F, d), "up": mat(L["up_q8"], F, d), "down": mat(L["down_q8"], d, F),
                        "n1": L["attn_norm"].astype(np.float64), "n2": L["ffn_norm"].astype(np.float64)} for L in sm.layers]
        self.cap, self.budget, self.recent = capacity or D["ctx"], budget, recent
        self.clear()

    def clear(self):
        D = self.D
        self.pos = 0
        # per layer and key / value head: rows held and the weight that they have received
        self.K = [[np.zeros((0, D["head_dim"])) for _ in range(D["n_kv_head"])] for _ in self.layers]
        self.V = [[np.zeros((0, D["head_dim"])) for _ in range(D["n_kv_head"])] for _ in self.layers]
        self.M = [[np.zeros(0) for _ in range(D["n_kv_head"])] for _ in self.layers]

    def held(self):
        return len(self.M[0][0])

    def cut(self, l):
        for h in range(self.D["n_kv_head"]):
            kept = plain_kept(self.M[l][h], len(self.M[l][h]), self.budget, self.recent)
            self.K[l][h], self.V[l][h], self.M[l][h] = self.K[l][h][kept], self.V[l][h][kept], self.M[l][h][kept]

    def rows(self, ids):
        """Rows of the ids at the next positions; logits after the last."""
        D, n = self.D, len(ids)
        hd, group = D["head_dim"], D["n_head"] // D["n_kv_head"]
        if n == 1 and self.held() + 1 > self.cap:
            for l in range(len(self.layers)):
                self.cut(l)
        freq = 10000.0 ** (-2.0 * np.arange(hd // 2) / hd)
        a = (self.pos + np.arange(n))[:, None] * freq

        def rotate(x):
            y = x.copy()
            y[..., 0::2] = x[..., 0::2] * np.cos(a)[:, None] - x[..., 1::2] * np.sin(a)[:, None]
            y[..., 1::2] = x[..., 0::2] * np.sin(a)[:, None] + x[..., 1::2] * np.cos(a)[:, None]
            return y
        rms = lambda v, w: v / np.sqrt((v * v).mean(-1, keepdims=True) + 1e-6) * w  # noqa: E731
        x = self.tok[ids]
        for l, L in enumerate(self.layers):
            h = rms(x, L["n1"])
            q, k = rotate((h @ L["wq"].T).reshape(n, -1, hd)), rotate((h @ L["wk"].T).reshape(n, -1, hd))
            v = (h @ L["wv"].T).reshape(n, -1, hd)
            out = np.zeros_like(q)
            for g in range(D["n_kv_head"]):
                self.K[l][g], self.V[l][g] = np.vstack([self.K[l][g], stands_for(k[:, g])]), np.vstack([self.V[l][g], stands_for(v[:, g])])
                held = len(self.K[l][g])
                self.M[l][g] = np.concatenate([self.M[l][g], np.zeros(n)])
                for j in range(group):
                    o, P = plain_attention(q[:, g * group + j], self.K[l][g], self.V[l][g], [held - n + i + 1 for i in range(n)], 1 / math.sqrt(hd))
                    out[:, g * group + j] = o
                    self.M[l][g] += P.sum(0)
            x = x + out.reshape(n, -1) @ L["wo"].T
            h = rms(x, L["n2"])
            gate = h @ L["gate"].T
            x = x + (gate / (1 + np.exp(-gate)) * (h @ L["up"].T)) @ L["down"].T
            if held > self.cap:
                self.cut(l)
        self.pos += n
        return rms(x[-1], self.norm) @ self.tok.T


def close(got, want):
    # f32 sums through a few layers: 1e-5 of the logits. A key or value within that of the border between two levels may fall to the
    # other side: one of some ten thousand, by a step of an eighth of its block, which moves a logit by less than a hundredth.
    assert np.abs(got - want).max() <= 1e-2 * np.abs(want).max()


@pytest.mark.gpu
@pytest.mark.parametrize("shape,prec", [("llama-mini", None), ("llama-hd64", None), ("qwen-odd", None), ("llama-mini", _lib.FC_Q_INT8)])
def test_prompt_and_steps_are_the_decoder_with_rounded_rows(shape, prec):
    sm = synth.llama_named(shape, seed=3, perturb=True)
    m = CudaLlama.from_synth(sm, prec=prec)
    if prec is not None:      # the packed weights are others: the f32 cache of the same model is what is near
        plain = None
    else:
        plain = Plain(sm)
    ids = synth.token_ids(5, 60, sm.dims["vocab"])
    cache, steps, wide = m.new_cache(kv4=True), m.new_cache(kv4=True), m.new_cache()
    for n in (40, 3):                                          # as a window, and id by id
        got = m.prime(ids[:n], cache)
        steps.clear()
        for t in ids[:n]:
            one = m.forward_one(t, steps)
        close(one, got)
        assert cache.pos() == cache.held() == n
        f32 = m.prime(ids[:n], wide)
        assert np.corrcoef(got, f32)[0, 1] > 0.9
        if plain:
            plain.clear()
            close(got, plain.rows(ids[:n]))
        for t in ids[n:n + 20]:
            got = m.forward_one(t, cache)
            if plain:
                close(got, plain.rows([t]))
    m.close()


@pytest.mark.gpu
@pytest.mark.parametrize("shape,n,capacity,budget,recent", [("llama-mini", 20, 24, 16, 4), ("llama-mini", 60, 32, 20, 20), ("llama-hd64", 90, 64, 33, 0), ("llama-mini", 5, 8, 2, 1)])
def test_a_small_cache_keeps_recent_and_attended_positions(shape, n, capacity, budget, recent):
    sm = synth.llama_named(shape, seed=4, perturb=True)
    m, plain = CudaLlama.from_synth(sm), Plain(sm, capacity, budget, recent)
    ids = synth.token_ids(6, n + 40, sm.dims["vocab"])
    cache = m.new_cache(kv4=True, capacity=capacity, budget=budget, recent=recent)
    got = m.prime(ids[:n], cache)
    if n < 8:
        for t in ids[:n]:
            want = plain.rows([t])
    else:
        want = plain.rows(ids[:n])
    close(got, want)
    assert cache.held() == plain.held() and cache.pos() == n
    for t in ids[n:]:
        close(m.forward_one(t, cache), plain.rows([t]))
        assert cache.held() == plain.held()
    assert cache.pos() == n + 40
    m.close()


@pytest.mark.gpu
@pytest.mark.parametrize("layout", [{}, {"capacity": 48, "budget": 30, "recent": 8}])
@pytest.mark.parametrize("prec", [None, _lib.FC_Q_INT4])
def test_generation_is_its_steps(layout, prec):
    """Eight tokens a graph, across evictions, again on the same cache and on the model's other one."""
    sm = synth.llama_named("llama-mini", seed=7, perturb=True)
    m = CudaLlama.from_synth(sm, prec=prec)
    ids = synth.token_ids(9, 30, sm.dims["vocab"])
    greedy = engine.sampling(temperature=0.0)
    cache, steps = m.new_cache(kv4=True, **layout), m.new_cache(kv4=True, **layout)
    logits = m.prime(ids, steps)
    want = []
    for _ in range(60):
        want.append(int(np.argmax(logits)))
        logits = m.forward_one(want[-1], steps)
    for _ in range(2):
        got, _ = m.generate(ids, 60, greedy, cache=cache)
        assert got.tolist() == want and cache.pos() == 90 and cache.held() == steps.held()
    f32, _ = m.generate(ids, 60, greedy, cache=m.new_cache())     # an f32 cache beside it is as ever
    again = m.new_cache()
    assert m.generate(ids, 60, greedy, cache=again)[0].tolist() == f32.tolist()
    m.close()


@pytest.mark.gpu
@pytest.mark.parametrize("shape,prec", [("llama-mini", None), ("llama-mini", _lib.FC_Q_INT8), ("llama-hd64", None)])
def test_a_failed_step_leaves_the_cache_as_it_was(shape, prec):
    """An id is lost on its way to a step: what the cache goes on with, evictions by received weight among it, is that of a cache
    which never failed, to the bit. Once it fails as the cache is full, once ahead of that, and in a generation that goes on behind it."""
    sm = synth.llama_named(shape, seed=8, perturb=True)
    m = CudaLlama.from_synth(sm, prec=prec)
    ids = synth.token_ids(10, 80, sm.dims["vocab"])
    layout = dict(capacity=24, budget=12, recent=3)
    sound, cache = m.new_cache(kv4=True, **layout), m.new_cache(kv4=True, **layout)
    failed = lambda call: fails_without_ids(call, _lib.FC_E_DIM)  # noqa: E731
    assert np.array_equal(m.prime(ids[:20], sound), m.prime(ids[:20], cache))
    for i, t in enumerate(ids[20:70]):
        if i in (2, 4, 5, 17):                                  # five to a full cache, then twelve a round
            for _ in range(60):                                 # what one of them would add is little
                failed(lambda: m.forward_one(ids[0], cache))
            assert cache.pos() == 20 + i
        assert np.array_equal(m.forward_one(t, sound), m.forward_one(t, cache)), i
        assert cache.held() == sound.held() and cache.pos() == sound.pos()
    # a prompt of six ids whose last is lost, and the eviction rounds of the tokens behind it
    small = dict(capacity=8, budget=3, recent=1)
    sound, cache = m.new_cache(kv4=True, **small), m.new_cache(kv4=True, **small)
    failed(lambda: m.generate(ids[:6], 30, engine.sampling(temperature=0.0), cache=cache))
    for t in ids[:5]:
        m.forward_one(t, sound)
    assert cache.pos() == cache.held() == 5
    for t in ids[30:50]:
        assert np.array_equal(m.forward_one(t, sound), m.forward_one(t, cache))
        assert cache.held() == sound.held()
    m.close()


@pytest.mark.gpu
@pytest.mark.parametrize("n", [20, 60])
def test_a_prompt_that_fails_leaves_an_empty_cache(n):
    """A wait of its products runs out: nothing of the prompt stays, evicted rows of one that is longer than the cache among it."""
    sm = synth.llama_named("llama-hd64", seed=8, perturb=True)
    m = CudaLlama.from_synth(sm)
    ids = synth.token_ids(10, 80, sm.dims["vocab"])
    layout = dict(capacity=24, budget=12, recent=3)
    sound, cache = m.new_cache(kv4=True, **layout), m.new_cache(kv4=True, **layout)
    for _ in range(2):
        fails_without_ids(lambda: m.prime(ids[:n], cache), _lib.FC_E_TIMEOUT)
        assert cache.pos() == cache.held() == 0
        sound.clear()
        for t in ids[:30]:
            assert np.array_equal(m.forward_one(t, sound), m.forward_one(t, cache))
            assert cache.held() == sound.held()
    assert np.array_equal(m.prime(ids[:n], sound), m.prime(ids[:n], cache))
    m.close()


@pytest.mark.gpu
def test_a_step_that_finds_no_memory_leaves_the_cache_at_the_last_one():
    """Sixteen heads on one: their weights take softmax statistics, from a pool that has nothing when the last step of a feed is captured."""
    sm = synth.SynthLlama(512, 256, 2, 16, 1, 32, 512, 128, seed=3, perturb=True)
    m, plain = CudaLlama.from_synth(sm), Plain(sm, 12, 7, 2)
    ids = synth.token_ids(4, 60, 512)
    layout = dict(capacity=12, budget=7, recent=2)
    sound, cache = m.new_cache(kv4=True, **layout), m.new_cache(kv4=True, **layout)
    m.forward_one(ids[0], cache, want_logits=False)            # the form of a feed's first steps
    _lib.lib().fc_debug_withhold_scratch(1)
    try:
        with pytest.raises(fcb.FerrumCudaError) as e:
            m.prime(ids[:5], cache)
        assert e.value.code == _lib.FC_E_CUDA
        with pytest.raises(fcb.FerrumCudaError):
            m.forward_one(ids[4], cache)
    finally:
        _lib.lib().fc_debug_withhold_scratch(0)
    assert cache.pos() == cache.held() == 4
    for t in ids[:4]:
        m.forward_one(t, sound, want_logits=False)
        plain.rows([t])
    for t in ids[4:40]:
        got = m.forward_one(t, cache)
        assert np.array_equal(got, m.forward_one(t, sound)) and cache.held() == sound.held()
        close(got, plain.rows([t]))
    assert m.generate(ids[:5], 40, engine.sampling(temperature=0.0), cache=cache)[0].tolist() == m.generate(ids[:5], 40, engine.sampling(temperature=0.0), cache=sound)[0].tolist()
    m.close()


def fails_without_ids(call, code):
    _lib.check(_lib.lib().fc_debug_set_wait_budget(200_000, 1))
    try:
        with pytest.raises(fcb.FerrumCudaError) as e:
            call()
    finally:
        _lib.check(_lib.lib().fc_debug_set_wait_budget(4_000_000_000, 0))
    assert e.value.code == code


def test_layouts_are_checked_before_a_device_is_used():
    assert _lib.lib().fc_llama_cache_create_kv4(None, 0, 0, 0, C.byref(C.c_void_p())) == _lib.FC_E_ARG
    assert _lib.lib().fc_llama_cache_held(None) == 0


@pytest.mark.gpu
def test_layouts_that_are_refused():
    m = CudaLlama.from_synth(synth.llama_named("llama-mini", seed=1))
    for layout, code in (({"capacity": 257}, _lib.FC_E_DIM), ({"capacity": -1}, _lib.FC_E_DIM), ({"capacity": 16}, _lib.FC_E_SHAPE),
                         ({"capacity": 16, "budget": 16}, _lib.FC_E_SHAPE), ({"capacity": 16, "budget": 8, "recent": 9}, _lib.FC_E_SHAPE),
                         ({"capacity": 16, "budget": 8, "recent": -1}, _lib.FC_E_SHAPE)):
        with pytest.raises(fcb.FerrumCudaError) as e:
            m.new_cache(kv4=True, **layout)
        assert e.value.code == code
    cache = m.new_cache(kv4=True, capacity=16, budget=8)
    with pytest.raises(fcb.FerrumCudaError) as e:               # the context is the model's, whatever the cache holds
        m.prime(np.zeros(257, np.int32), cache)
    assert e.value.code == _lib.FC_E_DIM
    narrow = CudaLlama.from_synth(synth.llama_named("llama-tiny", seed=1))
    with pytest.raises(fcb.FerrumCudaError) as e:               # heads of 16
        narrow.new_cache(kv4=True)
    assert e.value.code == _lib.FC_E_SHAPE
    m.close()
    narrow.close()


@pytest.mark.gpu
def test_a_serving_loop_of_the_operators():
    """Prompts with weights, an eviction to a smaller cache, steps on it and draws from their logits, on one stream."""
    rng = np.random.default_rng(12)
    S, heads, kv, dim, V, budget, recent = 3, 8, 2, 64, 900, 24, 6
    rows = [50, 31, 24]
    cap, room = max(rows), budget + 10
    big, small = kv4.Kv4Cache(S, kv, dim, cap), kv4.Kv4Cache(S, kv, dim, room)
    st = torch.cuda.Stream()
    s = C.c_void_p(st.cuda_stream)
    width = (heads + 2 * kv) * dim
    x, head = draws(rng, sum(rows), width), (rng.standard_normal((V, heads * dim)) / 16).astype(np.float32)
    xd, hd = dev(x), dev(head)
    out, mass, zero, lens = torch.empty((sum(rows), heads * dim), device="cuda"), torch.zeros((S, kv, cap), device="cuda"), ints([0] * S), ints(rows)
    left, mass2, kept = ints([0] * S), torch.zeros((S, kv, room), device="cuda"), torch.zeros((S, kv, budget), dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    k = 4 * heads * dim
    big.attend_dev(xd.data_ptr(), width, heads, zero.data_ptr(), out.data_ptr(), heads * dim, k_ptr=xd.data_ptr() + k, v_ptr=xd.data_ptr() + k + 4 * kv * dim, ldkv=width,
                   rows=rows, mass_ptr=mass.data_ptr(), stream=s)
    big.evict_dev(small, lens.data_ptr(), left.data_ptr(), budget, recent, mass.data_ptr(), mass2.data_ptr(), kept.data_ptr(), stream=s)
    # the oracle's caches, from the positions that were kept: the same but where weights tie to rounding
    K, V_ = [], []
    at = 0
    torch.cuda.synchronize()
    for i, n in enumerate(rows):
        xk = stands_for(x[at:at + n, heads * dim:(heads + kv) * dim].reshape(n, kv, dim))
        xv = stands_for(x[at:at + n, (heads + kv) * dim:].reshape(n, kv, dim))
        q = x[at:at + n, :heads * dim].astype(np.float64).reshape(n, heads, dim)
        for h in range(kv):
            got = np.zeros(n)
            for g in range(heads // kv):
                got += plain_attention(q[:, h * (heads // kv) + g], xk[:, h], xv[:, h], range(1, n + 1), dim ** -0.5)[1].sum(0)
            want = plain_kept(got, n, budget, recent)
            mine = kept[i, h, :min(n, budget)].tolist()
            other = sorted(set(want) ^ set(mine))
            assert not other or np.ptp(got[other]) < 1e-4
            K.append(xk[mine, h])
            V_.append(xv[mine, h])
        at += n
    params = torch.tensor([[0.9, 0.0, 0.95, 0.02]] * S).cuda()
    step_out, logits, token = torch.empty((S, heads * dim), device="cuda"), torch.empty((S, V), device="cuda"), torch.zeros(S, dtype=torch.int32, device="cuda")
    for step in range(10):
        y = draws(rng, S, width)
        yd, ud = dev(y), dev(rng.random(S).astype(np.float32))
        torch.cuda.synchronize()
        small.attend_dev(yd.data_ptr(), width, heads, left.data_ptr(), step_out.data_ptr(), heads * dim, k_ptr=yd.data_ptr() + k, v_ptr=yd.data_ptr() + k + 4 * kv * dim,
                         ldkv=width, mass_ptr=mass2.data_ptr(), stream=s)
        with torch.cuda.stream(st):
            torch.matmul(step_out, hd.T, out=logits)
            left += 1
        engine.sample_rows_dev(logits.data_ptr(), V, S, V, params.data_ptr(), ud.data_ptr(), token.data_ptr(), stream=s)
        torch.cuda.synchronize()
        o, lg = step_out.cpu().numpy(), logits.cpu().numpy()
        for i in range(S):
            for h in range(kv):
                c = i * kv + h
                K[c] = np.vstack([K[c], stands_for(y[i, (heads + h) * dim:(heads + h + 1) * dim])[None]])
                V_[c] = np.vstack([V_[c], stands_for(y[i, (heads + kv + h) * dim:(heads + kv + h + 1) * dim])[None]])
                for g in range(heads // kv):
                    a = (h * (heads // kv) + g) * dim
                    qq = y[i:i + 1, a:a + dim].astype(np.float64)
                    want = plain_attention(qq, K[c], V_[c], [len(K[c])], dim ** -0.5)[0][0]
                    tol = np.abs(V_[c]).max() * (2 * score_error(qq, K[c], dim ** -0.5) + 2.0 ** -20 + 66 * 2.0 ** -23)
                    assert np.abs(o[i, a:a + dim] - want).max() <= tol
            want, _, near = plain_draw(lg[i], 0.9, 0, 0.95, 0.02, float(ud[i]))
            assert token[i] == want or near < 1e-9
    assert left.tolist() == [min(n, budget) + 10 for n in rows]
