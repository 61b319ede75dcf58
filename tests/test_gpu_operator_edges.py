"""GPU: calls of the rotary, 4-bit cache and scoring operators at their edges, each against its definition in 64 bits or against torch's own manner."""
import pytest
import torch

from test_gpu_kv4 import check as check_attention, filled, levels
from test_gpu_long_context import build
from test_gpu_logprobs import TYPES, check as check_scores, gen
from ternainfer_b200.kv4 import KV4Cache, kv4_append, kv4_attend
from ternainfer_b200.rotary import rotary_table, rotate
from ternainfer_b200.scores import token_logprobs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,H,K", [(64, 8, 2), (128, 12, 1)])
def test_equal_shares_of_short_sequences_in_a_large_cache(lib, D, H, K):
    """So many places that keys are cut into equal shares whatever the lengths: each CTA finds its first sequence, head and block before it writes
    the query's fragments; again and again the same numbers."""
    B, L, n = 400 // K, 6016, 700
    cache = KV4Cache.empty(B, K, L, D)
    k, v = (torch.randn((B, n, K, D), generator=gen(i), device="cuda").to(torch.bfloat16) for i in (1, 2))
    kv4_append(cache, k, v, torch.zeros(1, dtype=torch.int64, device="cuda"))
    k, v = levels(k)[0], levels(v)[0]
    q = torch.randn((B, 1, H, D), generator=gen(3), device="cuda").to(torch.bfloat16)
    for low, high in ((0, n), (n - 3, n), (0, 2)):
        start = torch.randint(low, high, (B,), generator=gen(high), device="cuda")
        got = check_attention(q, cache, k, v, start)
        for _ in range(30):
            assert torch.equal(kv4_attend(q, cache, start), got)
    assert lib.ternaspmm_last_status() == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,size", [(16, 8192), (1500, 20000), (1500, 32000)])
def test_ties_between_a_rows_end_and_its_middle(lib, dtype, N, size):
    """Rows of several 4 KB at a warp each that end off a 16-byte boundary: of equal logits the lowest ids, whichever piece of the row they are in."""
    V = size // torch.finfo(dtype).bits * 8 - 3
    chunk = 4096 // torch.finfo(dtype).bits * 8
    base = (0.5 * torch.randn((N, V + 9), generator=gen(V), device="cuda")).clamp(-4, 4).to(dtype)
    t = torch.randint(0, V, (N,), generator=gen(1), device="cuda")
    for top in (1, 5, 20, 32):
        y = base.clone()
        for off in (0, 1, 6):
            x = y[:, off: off + V]
            x[:, V - 1] = 7.0
            x[:, V - 2] = 6.0
            x[:, chunk + 100: chunk + 103] = 7.0
            x[:, 50: 50 + 7 * (top - 1): 7] = 7.0
            check_scores(x, t, top)
    assert lib.ternaspmm_last_status() == 0


def test_targets_that_change_before_the_backward_pass(lib):
    """As with torch's own operators: an error, not the gradient of other tokens."""
    x = torch.randn((4, 6, 500), generator=gen(1), device="cuda", requires_grad=True)
    for t in (torch.randint(0, 500, (4, 6), generator=gen(2), device="cuda"), torch.randint(0, 500, (4, 12), generator=gen(3), device="cuda")[:, ::2]):
        want, = torch.autograd.grad(token_logprobs(x, t.clone()).logprob.sum(), x)
        r = token_logprobs(x, t, 2)
        assert torch.equal(torch.autograd.grad(r.logprob.sum(), x, retain_graph=True)[0], want)
        t[0, 0] = 7
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(r.logprob.sum(), x)


@pytest.mark.parametrize("layout,n", [("interleaved", 64), ("half", 64), ("half", 32), ("interleaved", 36), ("half", 36)])
def test_append_beyond_the_table(lib, layout, n):
    """A cache longer than the rotary table: a sequence with a token at a position that the table lacks is not written at all, and its queries are NaN."""
    B, T, K, D, L = 5, 3, 2, 64, 100
    table = rotary_table(D, L, rotary_dim=n, layout=layout)
    cache, *_ = filled(B, K, 128, D, 3)
    before = [t.clone() for t in cache._tensors()]
    q, k, v = torch.randn((B, T, 4 + 2 * K, D), generator=gen(4), device="cuda").to(torch.bfloat16).split([4, K, K], 2)
    # the last one has no token, and lies behind the table
    for counts, ok in ((None, [True, True, False, False, False]), ([3, 2, 2, 1, 0], [True, True, True, False, True])):
        start, c = torch.tensor([50, 97, 98, 100, 120], device="cuda"), None if counts is None else torch.tensor(counts, device="cuda")
        got = kv4_append(cache, k, v, start, c, q=q, table=table)
        assert lib.ternaspmm_last_status() == 1
        fine = torch.tensor(ok, device="cuda")
        for a, b in zip(cache._tensors(), before):
            assert torch.equal(a[~fine], b[~fine]) and not torch.equal(a[:2], b[:2])
        assert got[~fine, ..., :n].isnan().all()
        want, _ = rotate(q[:2], None, table, start[:2, None] + torch.arange(T, device="cuda"))
        assert torch.equal(got[:2], want)
        lib.ternaspmm_last_status()
        for b in range(2):                               # those that fit are there, without a number that is not finite
            at = slice(int(start[b]), int(start[b]) + (T if counts is None else counts[b]))
            assert cache.k_scales[b, :, at].isfinite().all() and not torch.equal(cache.v_codes[b, :, at], before[2][b, :, at])
        out = kv4_attend(got, cache, start, c)
        assert out[~fine].isnan().all() and out[:2].isfinite().all()
        for a, b in zip(cache._tensors(), before):
            a.copy_(b)
        lib.ternaspmm_last_status()
    start = torch.tensor([50, 97, 98, 100, 120], device="cuda")
    kv4_append(cache, k, v, start)                       # without a table every position of the cache is one
    assert lib.ternaspmm_last_status() == 0 and not torch.equal(cache.k_codes[4], before[0][4])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [300, 20000])
def test_gradient_of_a_target_outside_of_the_vocabulary(lib, dtype, V):
    """Its log probability is NaN, and so is the gradient through it; other rows, and the gradient through the entropy alone, are as they are."""
    x = torch.randn((4, V), generator=gen(V), device="cuda").to(dtype).requires_grad_()
    t, good = torch.tensor([5, V, -1, 2 ** 40], device="cuda"), torch.tensor([5, 0, -1, 0], device="cuda")
    w = torch.tensor([1.0, -0.5, 2.0, 0.25], device="cuda")
    want = torch.autograd.grad((token_logprobs(x, good).logprob * w).sum(), x)[0]
    assert lib.ternaspmm_last_status() == 0
    got = torch.autograd.grad((token_logprobs(x, t).logprob * w).sum(), x)[0]
    assert lib.ternaspmm_last_status() == 1
    assert got[[1, 3]].isnan().all() and torch.equal(got[[0, 2]], want[[0, 2]])
    entropy = [torch.autograd.grad((token_logprobs(x, y).entropy * w).sum(), x)[0] for y in (good, t)]
    assert torch.equal(*entropy) and entropy[0].isfinite().all()
    r = token_logprobs(x, t)                             # a program that takes the bad rows out
    got = torch.autograd.grad((torch.where(t < V, r.logprob, 0) * w).sum(), x)[0]
    assert torch.equal(got, torch.where((t < V)[:, None], want, 0))
    lib.ternaspmm_last_status()


@torch.inference_mode()
@pytest.mark.parametrize("fused", [False, True])
def test_positions_of_the_models_4_bit_cache(lib, fused):
    """Tokens at consecutive positions inside of the table, from any first one on; others are refused: NaN, status 1, caches as they were."""
    m = build(max_len=100, kv_bits=4, fused_glue=fused)
    tok = torch.randint(0, 1024, (2, 12), generator=gen(5), device="cuda")
    at = torch.arange(12, device="cuda")
    cache = m.make_cache(2, "cuda")
    whole = m(tok, cache, at)
    again = m.make_cache(2, "cuda")
    m(tok[:, :5], again, at[:5])
    m(tok[:, 5:], again, at[5:])
    assert all(torch.equal(a, b) for x, y in zip(cache[:1], again[:1]) for a, b in zip(x._tensors(), y._tensors())) and lib.ternaspmm_last_status() == 0
    held = [[t.clone() for t in c._tensors()] for c in cache]
    for pos in (at.flip(0), at + (at > 6), at * 0 + 3, at + 89, at - 1):
        out = m(tok, cache, pos)
        assert lib.ternaspmm_last_status() == 1 and out.isnan().all()
        assert all(torch.equal(a, b) for c, h in zip(cache, held) for a, b in zip(c._tensors(), h))
    for pos in (at[:1] + 100, at[:1] + 127, at[:1] - 1):
        out = m(tok[:, :1], cache, pos)
        assert lib.ternaspmm_last_status() == 1 and out.isnan().all()
        assert all(torch.equal(a, b) for c, h in zip(cache, held) for a, b in zip(c._tensors(), h))
    for pos in (at[:5], at[:, None], torch.arange(13, device="cuda")):
        with pytest.raises(ValueError):
            m(tok, cache, pos)
    assert torch.equal(m(tok, cache, at), whole) and lib.ternaspmm_last_status() == 0


@pytest.mark.parametrize("T,past", [(1, 300), (3, 40), (160, 2000)])
def test_attention_at_the_ends_of_the_scales_range(lib, T, past):
    """Scores that are nothing beside their softmax, and queries of zeros: the mean of what a row sees, keys that it does not see left out."""
    B, H, K, D = 2, 8, 2, 64
    cache, k, v = filled(B, K, past + T + 70, D, 5)
    start = torch.tensor([past, past // 2], device="cuda")
    q = torch.randn((B, T, H, D), generator=gen(6), device="cuda").to(torch.bfloat16)
    q[:, :, 1], q[:, :, 2] = 0, 2.0 ** -100
    for scale in (1e-10, 1e-13, 1e-25, 1e-37):
        check_attention(q, cache, k, v, start, scale=scale)
    check_attention(q, cache, k, v, start, window=33, scale=1e-30)
    cache.k_scales.zero_()                               # the largest scale and queries, and keys of zeros
    big = (q.double() * 2.0 ** 100).to(torch.bfloat16)
    check_attention(big, cache, k * 0, v, start, scale=1e6)
    assert lib.ternaspmm_last_status() == 0


def test_more_than_2_23_short_rows(lib):
    N, V = (1 << 23) + 9, 3
    x = torch.randn((N, V), generator=gen(1), device="cuda")
    t = torch.randint(-1, V, (N,), generator=gen(2), device="cuda")
    check_scores(x, t, 2)
    x.requires_grad_()
    got, = torch.autograd.grad(token_logprobs(x, t).logprob.sum(), x)
    tail = x.detach()[-5:].clone().requires_grad_()
    assert torch.equal(got[-5:], torch.autograd.grad(token_logprobs(tail, t[-5:]).logprob.sum(), tail)[0])
    assert lib.ternaspmm_last_status() == 0


def test_gradients_that_arrive_lazily_negated(lib):
    """Of one row: where torch hands the gradient of an imaginary part on as a view whose sign is a mark."""
    x = torch.randn((1, 200), generator=gen(1), device="cuda", requires_grad=True)
    r = token_logprobs(x, torch.tensor([3], device="cuda"))
    want, = torch.autograd.grad(r.entropy.sum(), x, retain_graph=True)
    z = (torch.complex(r.logprob, r.entropy).conj() * 1j).real                # the entropy itself
    assert torch.equal(z, r.entropy) and torch.equal(torch.autograd.grad(z.sum(), x)[0], want)


@pytest.mark.parametrize("window", [0, 70])
@pytest.mark.parametrize("T,past", [(200, 0), (160, 2000)])
def test_rows_whose_every_score_is_minus_infinity(lib, T, past, window):
    """Keys beyond fp16 among many tokens make NaN of the rows that see them, also where all scores are -inf; rows that see no key stay zero."""
    B, H, K, D = 2, 16, 2, 64
    cache = KV4Cache.empty(B, K, past + T, D)
    k = torch.full((B, past + T, K, D), 1e5, device="cuda", dtype=torch.bfloat16)
    kv4_append(cache, k, torch.ones_like(k), torch.zeros(B, dtype=torch.int64, device="cuda"))
    q = torch.full((B, T, H, D), -1.0, device="cuda", dtype=torch.bfloat16)
    start, counts = torch.tensor([past, 0], device="cuda"), torch.tensor([T, 0], device="cuda")
    out = kv4_attend(q, cache, start, counts, window=window)
    assert out[0].isnan().all() and not out[1].any()
    assert lib.ternaspmm_last_status() == 0


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_of_single_elements_do_not_matter(lib, dtype):
    """One sequence, token or head of a tensor of odd row lengths: what torch keeps as its stride there is no distance between anything."""
    table = rotary_table(64, 20)
    base = torch.randn(4000, generator=gen(1), device="cuda").to(dtype)
    pos = torch.tensor([7], device="cuda")
    for shape, strides in (((1, 1, 5, 64), (999, 77, 66, 1)), ((1, 1, 1, 64), (3, 5, 7, 1)), ((3, 1, 1, 64), (200, 1, 13, 1)), ((1, 1, 4, 64), (1, 1, 64, 1))):
        for offset in (0, 1, 2, 6, 8):
            x = base.as_strided(shape, strides, offset)
            for layout in ("interleaved", "half"):
                y = rotary_table(64, 20, layout=layout)
                assert torch.equal(rotate(x, x, y, pos)[1], rotate(x.clone(memory_format=torch.contiguous_format), None, y, pos)[0])
            if dtype != torch.bfloat16:
                continue
            B, _, K, D = shape
            start = torch.full((B,), 7, device="cuda")
            a, b = (KV4Cache.empty(B, K, 64, D) for _ in range(2))
            c = x.clone(memory_format=torch.contiguous_format)
            assert torch.equal(kv4_append(a, x, x, start, q=x, table=table), kv4_append(b, c, c, start, q=c, table=table))
            assert all(torch.equal(s, t) for s, t in zip(a._tensors(), b._tensors())) and torch.equal(kv4_attend(x, a, start), kv4_attend(c, b, start))
    assert lib.ternaspmm_last_status() == 0


def test_a_scale_that_fp32_does_not_hold(lib):
    cache, start = KV4Cache.empty(1, 1, 64, 64), torch.zeros(1, dtype=torch.int64, device="cuda")
    q = torch.ones((1, 1, 1, 64), device="cuda", dtype=torch.bfloat16)
    for scale in (1e-50, 0.0, -1.0, 1.1e6, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="scale"):
            kv4_attend(q, cache, start, scale=scale)
    assert not kv4_attend(q, cache, start, scale=1e-45).any() and lib.ternaspmm_last_status() == 0
