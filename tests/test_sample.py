"""Draws: tokens by given random numbers against the float64 oracle (gpu), refusals (CPU)."""

import ctypes as C

import numpy as np
import pytest
import torch

import spinf_serve_amd as sa
from oracle import sample as oracle_sample
from spinf_serve_amd import _lib


# ------------------------------------------------------------------------------------------------ refusals (CPU)
def test_draws_refuse_what_they_do_not_take(lib):
    x, u = torch.zeros((2, 8)), torch.zeros(2)
    with pytest.raises(RuntimeError):
        sa.sample_tokens(x, u)   # no CPU path
    for how in (dict(temperature=-1.0), dict(temperature=float("nan")), dict(top_p=-0.1), dict(min_p=float("nan")), dict(top_k=-3), dict(top_k=2.5)):
        with pytest.raises(ValueError):
            sa.sample_tokens(x, u, **how)


def test_a_top_k_of_any_size(lib):
    """a whole number, however large (more than there are: all); what is none is a ValueError as other settings are"""
    x, u = torch.zeros((2, 8)), torch.zeros(2)
    for k in (float("inf"), float("nan"), 2.5, -1, np.float32("inf")):
        with pytest.raises(ValueError):
            sa.sample_tokens(x, u, top_k=k)
    for k in (3.0, np.int64(7), 1 << 40, 10**30):
        with pytest.raises(RuntimeError):   # (no CPU path)
            sa.sample_tokens(x, u, top_k=k)


def test_the_c_entry_refuses_bad_arguments(lib):
    x = torch.zeros(64)
    need = C.c_int64()

    def args():
        a = _lib.SampleArgs()
        a.logits, a.ld, a.rows, a.vocab, a.u, a.token = x.data_ptr(), 8, 2, 8, x.data_ptr(), x.data_ptr()
        a.all_temperature, a.all_top_p = 1.0, 1.0
        a.workspace, a.workspace_bytes = x.data_ptr() // 16 * 16, 1 << 40
        return a

    assert lib.spinf_sample_workspace(C.byref(args()), C.byref(need)) == 0 and need.value > 0
    assert lib.spinf_sample_workspace(C.byref(args()), None) == -1
    for name, v in (("logits", None), ("u", None), ("token", None), ("workspace", None), ("workspace_bytes", 8), ("rows", -1), ("rows", 65536), ("vocab", 0), ("vocab", (1 << 22) + 1), ("ld", 7), ("dtype", 2),
                    ("all_temperature", -1.0), ("all_top_p", float("nan")), ("all_min_p", -0.5)):
        a = args()
        setattr(a, name, v)
        assert lib.spinf_sample(C.byref(a), None) == -1, name
    a = args()
    a.rows = 0
    assert lib.spinf_sample(None, None) == -1 and lib.spinf_sample(C.byref(a), None) == 0


@pytest.mark.gpu
def test_draws_refuse_tensors_before_any_launch(dev):
    x, u = torch.zeros((3, 40), device=dev), torch.zeros(3, device=dev)
    t = torch.ones(3, device=dev)
    for bad in (x.double(), x[0], x.t(), x[:, ::2], x.half()):
        with pytest.raises(ValueError):
            sa.sample_tokens(bad, u)
    for bad in (u[:2], u.half(), u.cpu(), torch.zeros(6, device=dev)[::2], u[:, None]):
        with pytest.raises(ValueError):
            sa.sample_tokens(x, bad)
    for bad in (dict(temperature=t.double()), dict(top_k=t), dict(top_p=t[:2]), dict(min_p=t.cpu()), dict(top_k=t.long())):
        with pytest.raises(ValueError):
            sa.sample_tokens(x, u, **bad)
    with pytest.raises(ValueError):
        sa.sample_tokens(torch.zeros((1, 40), device=dev).expand(3, 40), u)
    assert sa.sample_tokens(x[:0], u[:0]).shape == (0,)


# ------------------------------------------------------------------------------------------------ against the oracle
def logits(kind, rows, vocab, seed):
    g = np.random.default_rng(seed)
    x = 2.2 * g.standard_normal((rows, vocab))
    if kind == "peaked":
        for r in range(rows):
            at = g.integers(0, vocab, min(200, vocab))
            x[r, at] = 4 + 9 * g.random(len(at)) ** 2
    elif kind == "ties":
        x = np.floor(2 * x) / 2
    elif kind == "equal":
        x[:] = -3.25
    elif kind == "masked":
        x[g.random((rows, vocab)) < 0.95] = -np.inf
        x[0] = -np.inf
        x[-1] = -np.inf
        x[-1, vocab // 2] = 1.5
        if rows > 2:
            x[1, g.random(vocab) < 0.5] = np.nan
    elif kind == "wide":
        x *= 1000
    elif kind == "narrow":
        x *= 1e-4
    elif kind == "infinite":
        x[:, g.integers(0, vocab, 3)] = np.inf
        x[0] = -np.inf
    elif kind == "signs":   # zeros of either sign are equal
        x = np.where(g.random((rows, vocab)) < 0.5, -0.0, 0.0)
    elif kind == "largest":
        x[:] = np.where(x > 2, np.finfo(np.float32).max, np.where(x < -2, np.finfo(np.float32).min, x))
    return x


def check(dev, x, dtype, u, how, pad=0, u_dtype=torch.float64, doubt=None):
    rows, vocab = x.shape
    t = torch.from_numpy(x.astype(np.float32)).to(dtype)
    wide = torch.full((rows, vocab + pad), 99.0, dtype=dtype, device=dev)
    wide[:, :vocab] = t.to(dev)
    given = {k: torch.from_numpy(v).to(dev) if isinstance(v, np.ndarray) else v for k, v in how.items()}
    ud = torch.from_numpy(u).to(u_dtype).to(dev)
    token, prob = sa.sample_tokens(wide[:, :vocab], ud, **given, return_prob=True)
    values, un = t.double().numpy(), ud.double().cpu().numpy()
    bad = 0
    for r in range(rows):
        one = {k: float(np.float32(v[r] if isinstance(v, np.ndarray) else v)) for k, v in how.items()}
        one["top_k"] = int(one.get("top_k", 0))
        want, p, near = oracle_sample.draw(values[r], un[r], **one)
        if near > 1e-10:   # (nearer, the two orders of summing may fall on either side of a border)
            assert int(token[r]) == want, (r, one, un[r], int(token[r]), want)
            assert abs(float(prob[r]) - p) <= p * 2.0**-22 + 1e-30
        bad += near <= 1e-10
    assert bad <= (1 + rows // 20 if doubt is None else doubt)
    assert torch.equal(token, sa.sample_tokens(wide[:, :vocab], ud, **given))
    return token


HOW = [
    dict(), dict(temperature=0.7), dict(temperature=0.0), dict(top_k=1), dict(top_k=40, temperature=0.8), dict(top_p=0.9), dict(min_p=0.05), dict(top_p=0.999, temperature=1.5), dict(top_k=300, top_p=0.8, min_p=0.02),
    dict(top_k=1000, top_p=0.97), dict(min_p=1.0), dict(top_p=0.0), dict(top_p=1e-6), dict(min_p=1e-12), dict(top_k=1 << 29), dict(temperature=20.0, top_p=0.5), dict(temperature=0.01, top_k=3), dict(min_p=2.0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind,rows,vocab,pad", [("peaked", 5, 32000, 0), ("flat", 3, 16385, 3), ("ties", 4, 5000, 1), ("masked", 6, 20000, 0), ("flat", 2, 262144, 0), ("peaked", 40, 97, 0), ("flat", 3, 1, 0)])
def test_draws_against_the_oracle(dev, kind, rows, vocab, pad, dtype):
    g = np.random.default_rng(vocab)
    x = logits(kind, rows, vocab, vocab + 1)
    for how in HOW:
        check(dev, x, dtype, g.random(rows), how, pad)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["equal", "wide", "narrow", "infinite", "signs", "largest"])
def test_draws_from_extreme_logits(dev, kind):
    g = np.random.default_rng(3)
    x = logits(kind, 3, 20011, 9)
    for how in HOW:
        check(dev, x, torch.float32, g.random(3), how)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [20011, 9000])
def test_logits_near_the_lowest(dev, vocab):
    """the largest some T above the least finite number, masked ones beside them: 60 T below it there is no number"""
    g = np.random.default_rng(5)
    x = -np.finfo(np.float32).max * (1 - 0.01 * g.random((3, vocab)))
    x[g.random((3, vocab)) < 0.5] = -np.inf
    for t in (9e35, 2e35, 3e36):
        for how in HOW:
            check(dev, x, torch.float32, g.random(3), {**how, "temperature": t})


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["infinite", "masked", "largest", "flat"])
def test_draws_at_temperatures_of_any_size(dev, kind):
    """the largest that 32 bits hold, an infinite one (all finite logits weigh the same), and subnormal ones"""
    g = np.random.default_rng(4)
    x = logits(kind, 4, 20011, 7)
    for t in (3.4e38, float("inf"), 1e-38, 1e-45):
        for how in HOW:
            check(dev, x, torch.float32, g.random(4), {**how, "temperature": t})
    how = dict(temperature=np.array([np.inf, 1.0, np.inf, 3.4e38], np.float32), top_k=np.array([7, 0, 5000, 300], np.int32), top_p=np.array([1, 0.9, 0.7, 1], np.float32))
    check(dev, x, torch.float32, g.random(4), how)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["masked", "largest", "flat"])
def test_equal_weights_under_an_infinite_temperature(dev, kind):
    """all finite logits weigh the same: none is less likely than the likeliest, whatever min-p"""
    g = np.random.default_rng(4)
    x = logits(kind, 4, 20011, 7)
    for how in HOW:
        check(dev, x, torch.float32, g.random(4), {**how, "temperature": float("inf")})


@pytest.mark.gpu
def test_settings_of_every_row(dev):
    g = np.random.default_rng(8)
    rows = 96
    x = logits("peaked", rows, 50000, 4)
    x[7] = np.nan
    f = lambda *v: g.choice(np.array(v, np.float32), rows)  # noqa: E731
    how = dict(temperature=f(0, 0.5, 1, 1.4), top_k=g.choice(np.array([0, 1, 20, 50, 200, -1, 70000], np.int32), rows), top_p=f(1, 0.9, 0.3, 0.0, 2.0), min_p=f(0, 0, 0.1, 0.01))
    how["temperature"][3] = -1
    how["top_p"][4] = np.nan
    how["min_p"][5] = -0.1
    token = check(dev, x, torch.float32, g.random(rows), how)
    assert token[[3, 4, 5, 7]].tolist() == [-1] * 4


@pytest.mark.gpu
def test_random_numbers_at_the_ends(dev):
    x = logits("peaked", 6, 40000, 2)
    x[:, 0] = -np.inf
    u = np.array([0.0, 1.0, 1.5, -0.5, np.nan, 1 - 2.0**-53])
    for how in (dict(), dict(top_k=7), dict(top_p=0.6), dict(min_p=0.1)):
        for dt in (torch.float64, torch.float32):
            token = check(dev, x, torch.float32, u, how, u_dtype=dt)
            assert (token > 0).all()


@pytest.mark.gpu
def test_how_often_tokens_come(dev):
    """20,000 draws of one row: counts within 6 standard deviations of what the probabilities say"""
    x = torch.tensor([[1.0, 0.0, 2.0, -1.0, 0.5, -float("inf"), 1.5, 0.0]], device=dev)
    n = 20000
    u = torch.rand(n, generator=torch.Generator(device=dev).manual_seed(1), device=dev)
    got = sa.sample_tokens(x.repeat(n, 1), u, temperature=0.9, top_k=6, min_p=0.05)
    p = torch.softmax(x[0].double() / 0.9, 0)
    keep = torch.zeros(8, dtype=torch.bool, device=dev)
    keep[torch.sort(x[0], descending=True, stable=True)[1][:6]] = True
    p = torch.where(keep & (p >= 0.05 * p.max()), p, 0)
    p /= p.sum()
    count = torch.bincount(got, minlength=8).double()
    assert ((count - n * p).abs() <= 6 * (n * p * (1 - p)).sqrt() + 1e-9).all()


@pytest.mark.gpu
def test_graphs_streams_and_the_registered_operator(dev):
    x = torch.from_numpy(logits("peaked", 8, 40000, 2)).float().to(dev)
    u = torch.rand(8, device=dev)
    k = torch.full((8,), 30, dtype=torch.int32, device=dev)
    how = dict(temperature=0.9, top_k=k, top_p=0.95, return_prob=True)
    want = sa.sample_tokens(x, u, **how)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert all(torch.equal(a, b) for a, b in zip(sa.sample_tokens(x, u, **how), want))
    torch.cuda.synchronize()
    torch.library.opcheck(torch.ops.spinf.sample_tokens.default, (x, u, None, k, None, None, [0.9, 0, 0.95, 0.0], True), test_utils=("test_schema", "test_faketensor"))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        token, prob = sa.sample_tokens(x, u, **how)
    for i in range(3):
        u.copy_(torch.rand(8, generator=torch.Generator().manual_seed(i)))
        k.fill_(5 + 50 * i)
        graph.replay()
        torch.cuda.synchronize()
        e = sa.sample_tokens(x, u, **how)
        assert torch.equal(token, e[0]) and torch.equal(prob, e[1])
        torch.cuda.synchronize()


@pytest.mark.gpu
@pytest.mark.parametrize("base", [1e4, 1e7, 1e9, -1e9, 3e38])
def test_logits_whose_neighbours_lie_far_apart(dev, base):
    """numbers of 24 bits next to a large one: steps of 2^-10 to more than any temperature"""
    g = np.random.default_rng(6)
    x = np.full(9000, np.float32(base))
    for i in range(3):
        x[i::3] = np.nextafter(x[i::3], -np.inf) if i else x[i::3]
    x[2::3] = np.nextafter(x[2::3], np.float32(-np.inf))
    x[g.integers(0, 9000, 50)] = np.float32(base) - np.float32(abs(base) * 1e-3)
    x = x.astype(np.float64)[None].repeat(3, 0)
    for how in (dict(), dict(temperature=50.0), dict(top_p=0.4), dict(min_p=0.3), dict(top_k=4500, top_p=0.9)):
        check(dev, x, torch.float32, g.random(3), how)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["three values", "around zero", "one bin", "two heaps"])
def test_borders_among_many_tokens(dev, kind, dtype):
    """thousands of tokens in question: equal ones, ones of both signs, ones that share a bin, a border far below the largest"""
    rng = np.random.default_rng(len(kind))
    rows, vocab = 4, 40000
    x = {"three values": rng.integers(0, 3, (rows, vocab)) * 0.5, "around zero": rng.uniform(-1, 1, (rows, vocab)) * 0.3, "one bin": 3 + rng.uniform(0, 1, (rows, vocab)) * 0.01,
         "two heaps": np.where(rng.random((rows, vocab)) < 1e-3, 0.0, -40.0) + rng.uniform(0, 0.02, (rows, vocab))}[kind]
    x[1, rng.integers(0, vocab, 20000)] = -np.inf
    u = rng.random(rows)
    for how in (dict(top_k=5000), dict(top_k=19000), dict(top_p=0.37), dict(top_k=30000, top_p=0.8), dict(top_k=900, top_p=0.5), dict(top_k=3000, top_p=0.97, min_p=0.3), dict(top_p=0.6, temperature=0.05)):
        # (half of 900 equal weights is reached by 450 of them exactly: a border without a rounding's distance, in all rows)
        equal = how == dict(top_k=900, top_p=0.5) and (kind == "three values" or (kind == "one bin" and dtype == torch.bfloat16))
        token = check(dev, x, dtype, u, how, doubt=rows if equal else None)
        if equal:
            values = torch.from_numpy(x.astype(np.float32)).to(dtype).double().numpy()
            for r in range(rows):
                assert int(token[r]) in [oracle_sample.draw(values[r], u[r], top_k=900, top_p=0.5 + off)[0] for off in (-1e-9, 1e-9)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_chance_of_an_unlikely_token(dev, dtype):
    """the first token kept, drawn by u = 0, where it is some 10^-8 and 10^-12 of the whole"""
    rng = np.random.default_rng(2)
    x = rng.standard_normal((6, 20000))
    x[:, 3] = x.max(1) - np.array([10, 17, 18.5, 20, 25, 28])
    x[:, :3] = -np.inf
    for how in (dict(), dict(top_k=20000 - 3), dict(top_p=1.0, min_p=1e-14), dict(top_k=19000, temperature=1.1)):
        check(dev, x, dtype, np.zeros(6), how)


def reach(weights, p):
    """the first n of these whole numbers (largest first) hold p of their sum: n, and how far that border lies from its neighbours, in weights of the token at it; exact"""
    mass = np.cumsum(np.asarray(weights, object))
    num, den = float(np.float32(p)).as_integer_ratio()
    n = int(np.searchsorted(mass * den, num * mass[-1])) + 1
    over, under = mass[n - 1] * den - num * mass[-1], num * mass[-1] - (mass[n - 2] * den if n > 1 else 0)
    return n, float(min(over, under) / (weights[n - 1] * den))


ONE = 1 << 110   # what a weight of 1 is as a whole number


def weigh(z):
    """exp(z) as 64 bits of precision and more give it"""
    return int(np.ldexp(np.exp(np.longdouble(z)), 110))


# Borders far below the largest logit.  One token of weight 1 is the vocabulary's last, those of the tail are the first by index, so the kept ones are tokens 0 .. n - 2 and the last: u just below and
# just above what the n - 1 weigh tells n.  A tail token weighs 10^-13 (2^-43.3) and more of the whole.  What may move the border, in weights of such a token: weights are right to 2^-43 of
# themselves, which moves a border by (1 - p) / weight (at most 2^21) times that, 2^-22; p of the sum is a number of 64 bits, 2^-53 of the whole, 2^-9.  `reach` says how far it lies from the next.
@pytest.mark.gpu
@pytest.mark.parametrize("dtype,tail,temperature,top_k,top_p,vocab", [
    (torch.float32, -26.0, 1.0, 0, 0.9999995, 262144), (torch.float32, -26.0, 1.0, 0, 0.999999, 262144), (torch.bfloat16, -26.0, 1.0, 0, 0.9999995, 262144), (torch.float32, -13.5, 0.5, 0, 0.9999995, 262144),
    (torch.float32, -24.0, 1.0, 0, 0.9999995, 40000), (torch.float32, -26.5, 1.0, 0, 0.9999998, 151936), (torch.bfloat16, -30.0, 1.0, 0, 0.9999999, 1 << 22), (torch.float32, -28.0, 1.0, 0, 0.999999, 1 << 22),
    (torch.float32, -22.5, 1.0, 0, 0.99999, 262144), (torch.bfloat16, -20.0, 1.0, 0, 0.9999, 262144), (torch.float32, -26.0, 1.0, 200000, 0.9999995, 262144), (torch.float32, -12.0, 1.0, 150001, 0.7, 262144)])
def test_borders_of_top_p_far_below_the_largest(dev, dtype, tail, temperature, top_k, top_p, vocab):
    w, every = weigh(np.longdouble(tail) / np.longdouble(temperature)), top_k or vocab
    n, free = reach([ONE] + [w] * (every - 1), top_p)
    assert 5000 < n < every - 5000 and free > 2.0**-7
    x = torch.full((3, vocab), tail, dtype=dtype, device=dev)
    x[:, -1] = 0.0
    kept = ONE + (n - 1) * w
    u = np.array([(2 * n - 3) * w / (2 * kept), (2 * n - 1) * w / (2 * kept), w / (2 * kept)])
    token, prob = sa.sample_tokens(x, torch.from_numpy(u).to(dev), temperature=temperature, top_k=top_k, top_p=top_p, return_prob=True)
    assert token.tolist() == [n - 2, vocab - 1, 0], (n, free)
    for got, want in zip(prob.tolist(), (w / kept, ONE / kept, w / kept)):
        assert abs(got - want) <= want * 2.0**-22


@pytest.mark.gpu
@pytest.mark.parametrize("top_k,top_p", [(0, 0.9999995), (0, 0.9999998), (250000, 0.9999996)])
def test_borders_of_top_p_in_a_falling_tail(dev, top_k, top_p):
    """the same with a tail that falls by index from 24 to 30 below the largest: no two weights are equal"""
    vocab = 262144
    tail = np.linspace(-24, -30, vocab - 1).astype(np.float32)
    assert (np.diff(tail) < 0).all()
    weights = [ONE] + [weigh(z) for z in tail]
    every = top_k or vocab
    n, free = reach(weights[:every], top_p)
    assert 5000 < n < every - 5000 and free > 2.0**-7
    x = torch.from_numpy(np.concatenate([tail, np.zeros(1, np.float32)])).to(dev)[None].repeat(2, 1)
    before = sum(weights[1:n])   # the kept ones of the tail
    u = np.array([(2 * before - weights[n - 1]) / (2 * (ONE + before)), (2 * before + weights[n]) / (2 * (ONE + before))])
    token = sa.sample_tokens(x, torch.from_numpy(u).to(dev), top_k=top_k, top_p=top_p)
    assert token.tolist() == [n - 2, vocab - 1], (n, free)
