"""GPU: log probabilities of given tokens, entropy, alternatives and the gradient against log_softmax in 64 bits."""
import pytest
import torch

from ternainfer_b200.scores import token_logprobs

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def check(x, t, top):
    """Sums: every term is off by at most 2^-21 (exponential) and |x - m| 2^-23 (its argument), a thread adds up to n / 512 + 40 of them in
    fp32; log and the differences round a few times more."""
    got = token_logprobs(x, t, top)
    logp = torch.log_softmax(x.double(), -1)
    p = logp.exp()
    n = x.shape[-1] / 512 + 40
    rel = n * 2.0 ** -24 + 2.0 ** -20
    want = logp.gather(-1, t.clamp(0)[..., None])[..., 0].masked_fill(t < 0, 0)
    scale = torch.where(want.isfinite(), want.abs(), torch.zeros_like(want))
    assert torch.equal(got.logprob.isfinite(), want.isfinite())
    assert ((got.logprob.double() - want).nan_to_num(0, 0, 0).abs() <= rel + scale * 2.0 ** -22).all()
    h = -torch.special.xlogy(p, p).sum(-1)
    assert ((got.entropy.double() - h).abs() <= 4 * rel * (1 + h)).all(), (got.entropy.double() - h).abs().max()
    if top:
        v, i = torch.sort(x.float(), dim=-1, descending=True, stable=True)
        assert torch.equal(got.top_token, i[..., :top])
        want = logp.gather(-1, got.top_token)
        assert torch.equal(got.top_logprob.isneginf(), want.isneginf())
        assert ((got.top_logprob.double() - want).nan_to_num(0, 0, 0).abs() <= rel + want.nan_to_num(0, 0, 0).abs() * 2.0 ** -22).all()
    else:
        assert got.top_logprob is None and got.top_token is None
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,V", [(1, 1), (3, 2), (2, 7), (5, 33), (1, 511), (2, 512), (3, 513), (2, 1000), (7, 2049), (2, 4097), (300, 777), (3, 32000), (2, 128256), (1, 250001), (1, 1 << 19), (700, 20011)])
def test_logprobs(lib, dtype, N, V):
    g = gen(V)
    x = (3 * torch.randn((N, V), generator=g, device="cuda")).to(dtype)
    t = torch.randint(0, V, (N,), generator=g, device="cuda")
    for top in {0, 1, min(V, 5), min(V, 32)}:
        check(x, t, top)
    assert lib.ternaspmm_last_status() == 0


@pytest.mark.parametrize("dtype", TYPES)
def test_ties_bans_and_extremes(lib, dtype):
    """Equal logits, banned tokens, rows of one value, the type's largest and lowest, zeros of both signs."""
    V, g = 5000, gen(1)
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    x = torch.randn((12, V), generator=g, device="cuda")
    x[0] = 0.25
    x[1] = x[1].round()                                  # a few values, each thousands of times
    x[2, 100:4900] = float("-inf")
    x[3] = float("-inf")
    x[3, [7, 4000]] = 1.0                                # two tokens left
    x[4] = float("-inf")
    x[4, 4999] = -5.0                                    # one token left
    x = x.to(dtype)
    x[5] = low
    x[6, ::2], x[6, 1::2] = low, 3.0
    x[7, 17] = high
    x[8, ::2], x[8, 1::2] = 0.0, -0.0
    x[9] = torch.linspace(-5, 5, V, device="cuda").to(dtype)
    x[10] = x[9].flip(0)
    x[11] = torch.arange(V, device="cuda").remainder(512).to(dtype) / 64    # the same few threads hold all large values
    t = torch.randint(0, V, (12,), generator=g, device="cuda")
    t[3], t[4] = 7, 4999
    for top in (1, 2, 5, 32):
        check(x, t, top)
    one = token_logprobs(x[4:5], t[4:5], 3)
    # (one exponential, within 2^-22 of 1 relative to its argument, and a logarithm of it: nothing else is left of the sums)
    assert -2.0 ** -22 <= one.logprob.item() <= 0 and 0 <= one.entropy.item() <= 2.0 ** -21 and one.top_token[0].tolist() == [4999, 0, 1]


def test_rows_without_a_distribution(lib):
    V = 3000
    x = torch.zeros((4, V), device="cuda")
    x[0] = float("-inf")
    x[1, 5] = float("nan")
    x[2, 2500] = float("inf")
    t = torch.zeros(4, dtype=torch.int64, device="cuda")
    r = token_logprobs(x, t, 3)
    assert r.logprob[:3].isnan().all() and r.entropy[:3].isnan().all() and r.entropy[3].isfinite()
    assert r.top_token.tolist() == [[0, 1, 2], [5, 0, 1], [2500, 0, 1], [0, 1, 2]]
    assert lib.ternaspmm_last_status() == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [40, 300, 1031, 5000, 30000, 150000])
def test_rows_of_one_kind(lib, dtype, V):
    """More candidates than are kept: rows of NaN, of one value, of the lowest value, of -inf but for a few; a NaN and an infinity among others."""
    g = gen(V)
    x = torch.randn((9, V), generator=g, device="cuda").to(dtype)
    x[0], x[1], x[2], x[3] = float("nan"), 0.5, torch.finfo(dtype).min, float("-inf")
    x[3, 11], x[3, V - 1] = 1.0, 2.0
    x[4, V // 2] = float("nan")
    x[5, 0] = float("nan")
    x[6, [0, V - 1]] = float("inf")
    x[7, 3:] = x[7, 3]
    t = torch.zeros(9, dtype=torch.int64, device="cuda")
    for top in (1, 7, 32):
        got = token_logprobs(x, t, top)
        y = x.float()
        sort_key = torch.where(y.isnan(), torch.full_like(y, float("inf")), torch.where(y == float("inf"), torch.full_like(y, torch.finfo(torch.float32).max), y))
        order = torch.sort(sort_key, dim=-1, descending=True, stable=True)[1]
        assert torch.equal(got.top_token, order[:, :top])
    for r in (1, 2, 3, 7, 8):
        check(x[r: r + 1], t[r: r + 1] + (11 if r == 3 else 0), 5)
    assert got.logprob[[0, 4, 5, 6]].isnan().all() and got.entropy[[0, 4, 5, 6]].isnan().all()


@pytest.mark.parametrize("dtype", TYPES)
def test_many_short_rows(lib, dtype):
    """More rows than are at work at once, of lengths around those where a warp goes on to its next vectors; rows at any alignment."""
    g = gen(2)
    for N, V, step in ((5000, 131, 131), (4001, 255, 260), (700, 2050, 2051), (300, 8200, 8200), (64, 16391, 16400)):
        x = (3 * torch.randn((N, step), generator=g, device="cuda")).to(dtype)[:, :V]
        t = torch.randint(-1, V, (N,), generator=g, device="cuda")
        for top in (0, 20, 32):
            check(x, t, top)
        y = x.detach().clone().requires_grad_()
        got = token_logprobs(y, t)
        w = torch.randn(N, generator=g, device="cuda")
        grad, = torch.autograd.grad(got.logprob, y, w)
        p = torch.softmax(x.double(), -1)
        live = (t >= 0).double()[:, None]
        hot = torch.nn.functional.one_hot(t.clamp(0), V).double()
        want = (hot - p) * live * w[:, None].double()
        # p is off by 2^-18 of itself (its exponent holds up to 2^5, rounded three times, and the log of the sum); then one rounding
        eps = torch.finfo(dtype).eps / 2
        tiny = {torch.float16: 2.0 ** -25}.get(dtype, 0.0)
        assert ((grad.double() - want).abs() <= w.abs()[:, None].double() * live * p * 2.0 ** -18 * (1 + eps) + want.abs() * (eps + 2.0 ** -22) + tiny).all()
    assert lib.ternaspmm_last_status() == 0


def test_targets(lib):
    """No token, tokens outside of the vocabulary, any shape, rows apart from each other, targets of any strides."""
    g = gen(2)
    base = torch.randn((2, 6, 1003), generator=g, device="cuda").to(torch.bfloat16)
    t = torch.randint(0, 900, (2, 12), generator=g, device="cuda")[:, ::2]
    x = base[:, :, 1:901]
    got = check(x, t, 4)
    assert got.logprob.shape == (2, 6) and got.top_token.shape == (2, 6, 4)
    check(base.transpose(1, 2)[:, :500], torch.zeros((2, 500), dtype=torch.int64, device="cuda"), 3)
    check(base[:, :1].expand(2, 6, 1003), t, 3)
    t2 = t.clone()
    t2[0, 1], t2[1, 2] = -100, -1
    r = token_logprobs(x, t2)
    assert r.logprob[0, 1] == 0 and r.logprob[1, 2] == 0 and torch.equal(r.entropy, got.entropy) and lib.ternaspmm_last_status() == 0
    t2[0, 0] = 900
    r = token_logprobs(x, t2)
    assert r.logprob[0, 0].isnan() and r.logprob[0, 2:].equal(got.logprob[0, 2:]) and lib.ternaspmm_last_status() == 1
    assert token_logprobs(x[:, :0], t[:, :0], 2).top_token.shape == (2, 0, 2)
    assert token_logprobs(x[0, 0], t[0, 0]).logprob.shape == ()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,V", [(1, 1), (3, 65), (4, 1001), (2, 40000)])
def test_gradient(lib, dtype, N, V):
    g = gen(V)
    x = (2 * torch.randn((N, V), generator=g, device="cuda")).to(dtype)
    if V > 64:
        x[:, 50:60] = float("-inf")
    t = torch.randint(0, min(V, 50), (N,), generator=g, device="cuda")
    if N > 2:
        t[1] = -100
    gl, gh = torch.randn(N, generator=g, device="cuda"), torch.randn(N, generator=g, device="cuda")
    logp = torch.log_softmax(x.double(), -1)
    p, lp = logp.exp(), logp.clamp(min=-1e3)
    h = -(p * lp).sum(-1, keepdim=True)
    one = torch.nn.functional.one_hot(t.clamp(0), V).double()
    gt = gl.double().masked_fill(t < 0, 0)[:, None]
    n = 2.0 ** -24 * (V / 512 + 64) + 2.0 ** -20               # of a probability, as in check()
    for a, b in ((True, True), (True, False), (False, True)):
        leaf = x.clone().requires_grad_()
        r = token_logprobs(leaf, t, 1)
        loss = (r.logprob * gl).sum() * a + (r.entropy * gh).sum() * b if a and b else (r.logprob * gl).sum() if a else (r.entropy * gh).sum()
        got, = torch.autograd.grad(loss, leaf)
        want = a * gt * (one - p) - b * gh.double()[:, None] * p * (lp + h)
        size = a * gt.abs() * (one + p) + b * gh.double().abs()[:, None] * p * (lp.abs() + h + 1)
        tol = want.abs() * torch.finfo(dtype).eps / 2 + 8 * n * size + torch.finfo(dtype).tiny * torch.finfo(dtype).eps
        assert got.dtype == dtype and ((got.double() - want).abs() <= tol).all()
    if dtype == torch.float32 and V == 1001:                    # against differences
        d, e = torch.randn(x.shape, generator=g, device="cuda"), 1e-2
        def f(y):
            r = token_logprobs(y, t)
            return (r.logprob * gl + r.entropy * gh).double().sum()
        leaf = x.clone().requires_grad_()
        got, = torch.autograd.grad(f(leaf), leaf)
        slope = (f(x + e * d) - f(x - e * d)) / (2 * e)
        assert abs(slope - (got.double() * d.double()).sum()) < 2e-2 * got.double().norm() * d.double().norm() / V ** 0.5


@pytest.mark.parametrize("dtype", TYPES)
def test_gradient_of_fully_masked_rows(lib, dtype):
    """Rows of the type's lowest value alone are uniform, and so is their gradient; a row of -inf alone has none (NaN), its neighbours theirs."""
    V = 9000
    x = torch.full((3, V), torch.finfo(dtype).min, dtype=dtype, device="cuda")
    x[1], x[2, ::3] = float("-inf"), 5.0
    leaf = x.requires_grad_()
    r = token_logprobs(leaf, torch.full((3,), 6, device="cuda"))
    got, = torch.autograd.grad(r.logprob.sum(), leaf)
    want = -torch.stack([torch.full((V,), 1 / V), torch.full((V,), float("nan")), (torch.arange(V) % 3 == 0) * (3 / V)]).cuda().double()
    want[:, 6] += 1
    assert torch.equal(got.isnan(), want.isnan())
    # one exponential of ln V, in fp32: 2^-20 relative; then a rounding
    assert ((got.double() - want).nan_to_num(0).abs() <= want.nan_to_num(0).abs() * (2.0 ** -20 + torch.finfo(dtype).eps / 2) + torch.finfo(dtype).tiny).all()


def test_gradient_of_strided_and_broadcast_rows(lib):
    g = gen(5)
    base = torch.randn((4, 900), generator=g, device="cuda")
    t = torch.randint(0, 700, (4,), generator=g, device="cuda")
    for view in (lambda b: b[:, 3:703], lambda b: b[:1, :700].expand(4, 700)):
        a, b = base.clone().requires_grad_(), base.clone().double().requires_grad_()
        (token_logprobs(view(a), t).logprob.sum() + token_logprobs(view(a), t).entropy.sum()).backward()
        logp = torch.log_softmax(view(b), -1)
        (logp[torch.arange(4), t].sum() - (logp.exp() * logp).sum()).backward()
        assert ((a.grad.double() - b.grad).abs() <= 1e-5).all()


def test_streams_and_graphs(lib):
    g = gen(6)
    x = torch.randn((5, 20000), generator=g, device="cuda")
    t = torch.randint(0, 20000, (5,), generator=g, device="cuda")
    want = token_logprobs(x, t, 5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = token_logprobs(x, t, 5)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = token_logprobs(x, t, 5)
    x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(out, token_logprobs(x, t, 5)))


@pytest.mark.parametrize("N,V", [(17000, 128256), (1100000, 2000)])
def test_offsets_beyond_32_bits(lib, N, V):
    """More than 2^31 logits: the last rows give what they give alone, the gradient included."""
    x = torch.empty((N, V), device="cuda", dtype=torch.bfloat16).normal_(generator=gen(1))
    assert x.numel() > 1 << 31
    t = torch.randint(0, V, (N,), generator=gen(2), device="cuda")
    w = torch.randn(N, generator=gen(3), device="cuda")
    x.requires_grad_()
    r = token_logprobs(x, t, 4)
    grad, = torch.autograd.grad(r.logprob, x, w)
    y = x.detach()[-3:].clone().requires_grad_()
    alone = check(y.detach(), t[-3:], 4)
    want, = torch.autograd.grad(token_logprobs(y, t[-3:]).logprob, y, w[-3:])
    # (another number of rows may be summed in another order: both are within check()'s bound)
    bound = 2 * ((V / 512 + 40) * 2.0 ** -24 + 2.0 ** -20) + alone.logprob.abs() * 2.0 ** -21
    assert ((r.logprob[-3:] - alone.logprob).abs() <= bound).all() and torch.equal(r.top_token[-3:], alone.top_token)
    assert ((grad[-3:].float() - want.float()).abs() <= want.float().abs() * 2.0 ** -7 + w[-3:, None].abs() * 2.0 ** -126).all()
    assert lib.ternaspmm_last_status() == 0


def test_refusals(lib):
    x, t = torch.zeros((2, 50), device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda")
    for bad in (dict(logits=x.double()), dict(targets=t.int()), dict(targets=t[:1]), dict(targets=t.cpu()), dict(top=33), dict(top=-1), dict(logits=x[:, :0]),
                dict(logits=x[:, :4], top=5), dict(logits=x.cpu())):
        with pytest.raises((ValueError, RuntimeError)):
            token_logprobs(**{**dict(logits=x, targets=t), **bad})
