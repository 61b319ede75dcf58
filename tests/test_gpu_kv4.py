"""GPU: the 4-bit key / value cache - what is written, what it stands for, attention over it - against plain forms in 64 bits."""
import math

import pytest
import torch

from ternainfer_b200.kv4 import KV4Cache, kv4_append, kv4_attend, kv4_read
from ternainfer_b200.rotary import rotary_table, rotate

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def levels(x):
    """What a group of 32 stands for (float64) and its scale: the definition, without the cache's layout."""
    g = x.double().unflatten(-1, (-1, 32))
    big = g.abs().amax(-1, keepdim=True)
    scale = (torch.where((g == big).any(-1, keepdim=True), big, -big) / -8).half().double()
    # (quotients in fp32, as the kernel takes them; a value a hair from the middle of two codes is either)
    code = torch.where(scale == 0, torch.zeros_like(g), (g.float() / scale.float()).round().double().clamp(-8, 7))
    return (code * scale).flatten(-2), scale.flatten(-2)


def filled(B, K, L, D, seed, spread=1.0):
    """A cache full of normal values, by the kernel; keys and values in float64."""
    g = gen(seed)
    cache = KV4Cache.empty(B, K, L, D)
    k, v = ((torch.randn((B, cache.max_len, K, D), generator=g, device="cuda") * s).to(torch.bfloat16) for s in (spread, 1.0))
    kv4_append(cache, k, v, torch.zeros(B, dtype=torch.int64, device="cuda"))
    return cache, levels(k)[0], levels(v)[0]


def attention(q, k, v, start, counts, window, scale):
    """float64 result and a bound of its error, q [B, T, H, D], k, v [B, L, K, D]."""
    B, T, H, D = q.shape
    L, K = k.shape[1:3]
    at = start[:, None] + torch.arange(T, device=q.device)
    key = torch.arange(L, device=q.device)
    sees = (key <= at[..., None]) & (key < (start + counts)[:, None, None])
    if window:
        sees &= key > at[..., None] - window
    kk, vv = (torch.where((key < (start + counts)[:, None])[..., None, None], t, torch.zeros_like(t)).repeat_interleave(H // K, 2) for t in (k, v))
    s = torch.einsum("bthd,blhd->bhtl", q.double(), kk) * scale
    s = s.masked_fill(~sees[:, None], -math.inf)
    p = torch.softmax(s, -1).nan_to_num(0.0)
    out = torch.einsum("bhtl,blhd->bthd", p, vv)
    # The result is rounded to bf16: 2^-8.  Probabilities are rounded to fp16, and so are their products with the scales: 2^-11 of each
    # term twice, 2^-10 + 2^-22 together, and 2^-13 for exponentials and sums; below 2^-14 of the largest
    # scale by up to 2^-25 of it, times |code - 8| <= 8.  Scores: fp32 sums of exact products, 128 of them, then a few roundings:
    # 2^-16 of sum |q||k| each at most, as an exponent.  The two accumulators of a value run over codes up to 15 and over the offset of 8, so they
    # are up to 15 / 8 of the largest value where the result may be next to nothing: each MMA, one for each of at most n / 16 + 1 groups
    # of keys that a result goes through, may cut off a last place of both, 2 * 15 / 8 * 2^-23 < 2^-21 of the largest value.
    size = torch.einsum("bhtl,blhd->bthd", p, vv.abs())
    top = vv.abs().amax((1, 3))[:, None, :, None]
    n = float(counts.max() + start.max()) + 1
    q_size = (q.double().abs().amax(-1) * q.shape[-1]).permute(0, 2, 1) * kk.abs().amax((1, 3))[:, :, None] * scale
    lost = size * (2.0 ** -10 + 2.0 ** -13) + top * (n * 2.0 ** -24 * 2 + (n / 16 + 1) * 2.0 ** -21) + \
        (q_size * 2.0 ** -20).permute(0, 2, 1)[..., None] * size
    if T > 1:
        # Calls of many tokens round keys and values to fp16: 2^-11 of every product |q||k|, an exponent of the probability and of their sum, and
        # 2^-11 of every value.
        s_abs = (torch.einsum("bthd,blhd->bhtl", q.double().abs(), kk.abs()) * scale).masked_fill(~sees[:, None], 0).amax(-1)
        lost = lost + size * (2.0 ** -11 + 2.0 ** -10 * s_abs.permute(0, 2, 1)[..., None])
    # What is rounded to bf16 is the result with those errors: |r(out + e) - out| <= |e| + 2^-8 |out + e| <= lost + 2^-8 (|out| + lost)
    return out, lost + (out.abs() + lost) * 2.0 ** -8


def check(q, cache, k, v, start, counts=None, window=0, scale=None):
    B, T = q.shape[:2]
    got = kv4_attend(q, cache, start, counts, window=window, scale=scale)
    st = start.expand(B)
    out, tol = attention(q, k, v, st, torch.full_like(st, T) if counts is None else counts, window, q.shape[-1] ** -0.5 if scale is None else scale)
    err = (got.double() - out).abs()
    assert (err <= tol).all(), f"{(err - tol).max().item()} beyond, largest error {err.max().item()}"
    assert torch.equal(kv4_attend(q, cache, start, counts, window=window, scale=scale), got)
    return got


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,T,K", [(1, 1, 1), (3, 1, 5), (2, 37, 2), (1, 130, 3)])
def test_append_and_read(lib, D, B, T, K):
    g = gen(D + T)
    cache = KV4Cache.empty(B, K, T + 70, D)
    qkv = torch.randn((B, T, 3 * K, D), generator=g, device="cuda").to(torch.bfloat16)
    qkv[0, 0, 0, :32] = 0                                           # a group of zeros
    qkv[0, 0, 0, 32] = 300.0                                        # one value far from the others
    k, v = qkv[:, :, :K], qkv[:, :, K: 2 * K]
    start = torch.randint(0, 70, (B,), generator=g, device="cuda")
    assert kv4_append(cache, k, v, start) is None
    for got, x in zip(kv4_read(cache, start, T), (k, v)):
        assert torch.equal(got, levels(x)[0].to(torch.bfloat16))
    # everything else is as it was
    at = torch.zeros((B, cache.max_len), dtype=torch.bool, device="cuda")
    at.scatter_(1, start[:, None] + torch.arange(T, device="cuda"), True)
    for t in (cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales):
        assert not t.transpose(1, 2)[~at].any() and (t.transpose(1, 2)[at].float().abs().sum() > 0)
    assert lib.ternaspmm_last_status() == 0


@pytest.mark.parametrize("layout,n", [("interleaved", 128), ("half", 128), ("half", 64), ("interleaved", 40), ("half", 36)])
def test_append_rotates(lib, layout, n):
    """Rotated in the same launch as by rotate() and an append after it, bit for bit; one start for all sequences."""
    B, T, H, K, D = 3, 9, 8, 2, 128
    g = gen(n)
    qkv = torch.randn((B, T, H + 2 * K, D), generator=g, device="cuda").to(torch.bfloat16)
    q, k, v = qkv[:, :, :H], qkv[:, :, H: H + K], qkv[:, :, H + K:]
    table = rotary_table(D, 128, rotary_dim=n, layout=layout)
    start = torch.tensor([50], device="cuda")
    a, b = KV4Cache.empty(B, K, 64, D), KV4Cache.empty(B, K, 64, D)
    got = kv4_append(a, k, v, start, q=q, table=table)
    want_q, want_k = rotate(q, k, table, start + torch.arange(T, device="cuda"))
    assert kv4_append(b, want_k, v, start.expand(B).contiguous()) is None
    assert torch.equal(got, want_q)
    for n in ("k_codes", "k_scales", "v_codes", "v_scales"):
        assert torch.equal(getattr(a, n), getattr(b, n))
    assert kv4_append(a, k, v, start, table=table) is None and torch.equal(a.k_codes, b.k_codes)


def test_padded_batches(lib):
    B, T, K, D = 4, 6, 2, 64
    g = gen(5)
    cache = KV4Cache.empty(B, K, 64, D)
    for t in (cache.k_codes, cache.v_codes):
        t.fill_(0x5a)
    old = cache.k_codes.clone()
    k, v = (torch.randn((B, T, K, D), generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    start, counts = torch.tensor([0, 58, 60, 64], device="cuda"), torch.tensor([6, 3, 0, 0], device="cuda")
    q = torch.randn((B, T, 4, D), generator=g, device="cuda").to(torch.bfloat16)
    kv4_append(cache, k, v, start, counts)
    got_k, got_v = kv4_read(cache, start, T, counts)
    live = torch.arange(T, device="cuda") < counts[:, None]
    assert torch.equal(got_k, levels(k)[0].to(torch.bfloat16) * live[..., None, None]) and torch.equal(got_v[live], levels(v)[0].to(torch.bfloat16)[live])
    assert torch.equal(cache.k_codes[1, :, 61:], old[1, :, 61:]) and torch.equal(cache.k_codes[2:], old[2:])
    assert lib.ternaspmm_last_status() == 0
    # a query behind its sequence's last token sees what is there; one of a sequence that holds nothing is zero
    out = kv4_attend(q, cache, torch.zeros(4, dtype=torch.int64, device="cuda"), counts)
    assert not out[2:].any() and out[:2].isfinite().all()
    assert lib.ternaspmm_last_status() == 0


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,K", [(1, 1), (5, 5), (20, 5), (16, 2), (18, 2), (33, 3)])
@pytest.mark.parametrize("B,past,L", [(1, 0, 64), (2, 1, 64), (1, 15, 64), (3, 63, 64), (1, 64, 128), (2, 333, 400), (1, 2000, 2048)])
def test_attend_one_token(lib, D, H, K, B, past, L):
    cache, k, v = filled(B, K, L, D, past)
    q = torch.randn((B, 1, H, D), generator=gen(past + H), device="cuda").to(torch.bfloat16) * 1.5
    check(q, cache, k, v, torch.full((B,), past, device="cuda"))
    assert lib.ternaspmm_last_status() == 0


@pytest.mark.parametrize("D,H,K", [(128, 20, 5), (64, 8, 8), (128, 6, 2), (128, 17, 1)])
@pytest.mark.parametrize("B,T,past", [(1, 2, 0), (2, 5, 11), (1, 17, 0), (1, 64, 64), (2, 100, 77), (1, 333, 200), (1, 128, 0), (3, 129, 1000), (2, 700, 63)])
def test_attend_several_tokens(lib, D, H, K, B, T, past):
    cache, k, v = filled(B, K, past + T + 20, D, past + T, spread=2.0)
    qkv = torch.randn((B, T, H + 2 * K, D), generator=gen(T), device="cuda").to(torch.bfloat16)
    check(qkv[:, :, :H], cache, k, v, torch.tensor([past], device="cuda"))


@pytest.mark.parametrize("window", [1, 2, 15, 16, 17, 100, 5000])
@pytest.mark.parametrize("T", [1, 3, 70])
def test_attend_window_and_ragged(lib, window, T):
    B, H, K, D = 5, 8, 2, 128
    cache, k, v = filled(B, K, 640, D, T)
    q = torch.randn((B, T, H, D), generator=gen(window), device="cuda").to(torch.bfloat16)
    start = torch.tensor([0, 5, 130, 400, 640 - T], device="cuda")
    check(q, cache, k, v, start, window=window)
    check(q, cache, k, v, start, counts=torch.tensor([T, T // 2, 0, T, 1], device="cuda"), window=window)


@pytest.mark.parametrize("D,H,K,T", [(128, 8, 2, 1), (64, 5, 5, 1), (128, 12, 1, 1), (128, 4, 2, 3), (64, 3, 1, 5)])
def test_attend_sequences_of_all_lengths(lib, D, H, K, T):
    """Caches large enough for the work to be cut across sequences: empty ones, one key, whole tiles and ragged ones beside each other; less work
    than there are CTAs; windows; some outside of the cache."""
    B, L = 40, 8192 // K
    cache, k, v = filled(B, K, L, D, T)
    q = torch.randn((B, T, H, D), generator=gen(H), device="cuda").to(torch.bfloat16)
    g = gen(12)
    full = torch.full((B,), T, device="cuda")
    ragged = torch.randint(0, L - T + 1, (B,), generator=g, device="cuda")
    ragged[[0, 7, 8, 39]], ragged[3], ragged[4], ragged[20] = 0, 31, 32, L - T
    counts = full.clone()
    counts[[1, 7, 8, 30]] = 0
    empty = torch.zeros_like(ragged)
    one = empty.clone()
    one[11] = min(2000, L - 9)                # (within every one of these caches)
    for start, c, window in ((ragged, None, 0), (ragged, counts, 0), (ragged, None, 100), (empty, None, 0), (empty, empty, 0), (one, counts, 0), (empty + L - T, None, 0)):
        check(q, cache, k, v, start, counts=c, window=window)
    assert lib.ternaspmm_last_status() == 0
    bad = ragged.clone()
    bad[[5, 39]] = torch.tensor([cache.max_len, -1], device="cuda")      # (the capacity: L rounded up)
    out = kv4_attend(q, cache, bad)
    assert out.isnan().flatten(1).all(1).nonzero().flatten().tolist() == [5, 39] and lib.ternaspmm_last_status() == 1
    good = torch.ones(B, dtype=torch.bool, device="cuda")
    good[[5, 39]] = False
    ref, tol = attention(q[good], k[good], v[good], bad[good], full[good], 0, D ** -0.5)
    assert ((out[good].double() - ref).abs() <= tol).all()


def test_attend_long_cache(lib):
    """One sequence, more keys than any split takes in one go; the last keys alone decide, then the first."""
    B, H, K, D, L = 1, 8, 2, 128, 70000
    cache, k, v = filled(B, K, L, D, 9)
    q = torch.randn((B, 1, H, D), generator=gen(8), device="cuda").to(torch.bfloat16)
    start = torch.tensor([L - 1], device="cuda")
    check(q, cache, k, v, start)
    for at in (0, 1, L - 2, L - 1):
        peak = (k[:, at].repeat_interleave(H // K, 1) * 8).to(torch.bfloat16)[:, None]
        check(peak, cache, k, v, start)


def test_attend_values_of_any_size(lib):
    """Scales far apart among tokens and groups, queries and keys of any size; scores that leave one key."""
    B, H, K, D, L = 1, 4, 1, 128, 256
    g = gen(10)
    for k_size, v_size, q_size in ((1e-3, 1e-2, 1e3), (100.0, 1e3, 1e-2), (1.0, 1.0, 30.0), (1.0, 1.0, 0.0), (1e-2, 1.0, 1e-30)):
        cache = KV4Cache.empty(B, K, L, D)
        k, v = (torch.randn((B, L, K, D), generator=g, device="cuda") * s * 4 ** torch.randn((B, L, K, 1), generator=g, device="cuda") for s in (k_size, v_size))
        k, v = k.to(torch.bfloat16), v.to(torch.bfloat16)
        kv4_append(cache, k, v, torch.zeros(1, dtype=torch.int64, device="cuda"))
        q = (torch.randn((B, 1, H, D), generator=g, device="cuda") * q_size).to(torch.bfloat16)
        check(q, cache, levels(k)[0], levels(v)[0], torch.tensor([L - 1], device="cuda"))
        check(q, cache, levels(k)[0], levels(v)[0], torch.tensor([L - 9], device="cuda"), scale=0.01)


@pytest.mark.parametrize("T", [1, 40])
def test_what_is_not_seen_does_not_matter(lib, T):
    """NaN and infinite scales in rows that hold no token, and in tokens that a query does not see."""
    B, H, K, D, L = 2, 8, 2, 128, 192
    cache, k, v = filled(B, K, L, D, 3)
    q = torch.randn((B, T, H, D), generator=gen(4), device="cuda").to(torch.bfloat16)
    start = torch.tensor([20, 77], device="cuda")
    want = check(q, cache, k, v, start)
    for b in range(B):
        end = int(start[b]) + T
        cache.k_scales[b, :, end:], cache.v_scales[b, :, end:] = float("nan"), float("inf")
        cache.k_codes[b, :, end:], cache.v_codes[b, :, end:] = 255, 255
    assert torch.equal(kv4_attend(q, cache, start), want)
    if T > 1:
        cache.v_scales[0, :, 20 + T - 1] = float("nan")            # the last token's value: only its own query sees it
        cache.k_scales[1, 0, 77 + T - 1] = float("nan")
        out = kv4_attend(q, cache, start)
        assert torch.equal(out[0, :-1], want[0, :-1]) and out[0, -1].isnan().all()
        assert torch.equal(out[1, :-1], want[1, :-1]) and out[1, -1, :4].isnan().all() and torch.equal(out[1, -1, 4:], want[1, -1, 4:])
    cache.v_scales[0, 1, 0, 2] = float("nan")                      # one group of one key, seen by all
    out = kv4_attend(q, cache, start)
    assert out[0, :, 4:, 64:96].isnan().all() and out[0, :-1, 4:, :64].isfinite().all() and out[0, :-1, :4].isfinite().all()


def test_values_beyond_fp16_among_many_tokens(lib):
    """Scales that make values beyond 65504: the rows that see one have NaN in its group, the others their results."""
    B, T, H, K, D = 1, 200, 4, 1, 128
    cache, k, v = filled(B, K, T, D, 3)
    q = torch.randn((B, T, H, D), generator=gen(4), device="cuda").to(torch.bfloat16)
    start = torch.zeros(1, dtype=torch.int64, device="cuda")
    want = check(q, cache, k, v, start)
    cache.v_scales[0, 0, 70, 1], cache.v_scales[0, 0, 150, 3] = 60000.0, float("-inf")
    out = kv4_attend(q, cache, start)
    lost = torch.zeros((T, D), dtype=torch.bool, device="cuda")
    lost[70:, 32:64], lost[150:, 96:] = True, True
    assert torch.equal(out.isnan(), lost[None, :, None].expand_as(out)) and torch.equal(out[0][:, :, :32], want[0][:, :, :32])
    assert torch.equal(out[0].masked_fill(lost[:, None], 0), want[0].masked_fill(lost[:, None], 0))


@pytest.mark.parametrize("D,H,K", [(128, 20, 5), (64, 8, 2), (128, 3, 3)])
@pytest.mark.parametrize("B,T,past,window", [(1, 120, 3000, 0), (2, 257, 1500, 0), (8, 33, 700, 0), (1, 130, 2900, 1), (2, 200, 1000, 64), (1, 300, 2700, 65), (3, 90, 1700, 1000), (1, 1000, 0, 300)])
def test_attend_keys_in_parts(lib, D, H, K, B, T, past, window):
    """Many tokens over long caches: the keys of a tile of rows in parts, with parts that no row or some rows see; padded batches; sequences that
    are shorter than the cache."""
    cache, k, v = filled(B, K, past + T + 20, D, past + T)
    q = torch.randn((B, T, H, D), generator=gen(T), device="cuda").to(torch.bfloat16)
    start = torch.tensor([past, 5, 0, 64, 63, 650, past, 1][:B], device="cuda")
    check(q, cache, k, v, start, window=window)
    check(q, cache, k, v, start, counts=torch.tensor([T - 1, 1, 0, T, T // 2, 3, T, 0][:B], device="cuda"), window=window)
    assert lib.ternaspmm_last_status() == 0
    start = start.clone()
    start[0] = cache.max_len - T + 1
    out = kv4_attend(q, cache, start, window=window)
    assert out[0].isnan().all() and out[1:].isfinite().all() and lib.ternaspmm_last_status() == 1


@pytest.mark.parametrize("window", [0, 30, 500])
@pytest.mark.parametrize("B,past", [(1, 100), (1, 2300), (2, 2500)])
def test_bad_scales_among_many_tokens(lib, window, B, past):
    """Scales that are NaN, infinite or make values beyond 65504: only the rows whose window holds one lose its group; a NaN key loses the row."""
    T, H, K, D = 300, 8, 2, 128
    cache, k, v = filled(B, K, past + T + 40, D, 3)
    q = torch.randn((B, T, H, D), generator=gen(4), device="cuda").to(torch.bfloat16)
    start = torch.full((B,), past, dtype=torch.int64, device="cuda")
    want = check(q, cache, k, v, start, window=window)
    at = past + torch.arange(T, device="cuda")
    lost = torch.zeros((B, T, H, D), dtype=torch.bool, device="cuda")
    for b, head, key, group, value in ((0, 1, past + 70, 1, 60000.0), (0, 1, past + 20, 1, float("nan")), (0, 0, past - 20, 3, float("-inf")), (B - 1, 1, past + T - 1, 0, float("nan")),
                                       (0, 0, past + T, 2, float("nan"))):
        cache.v_scales[b, head, key, group] = value
        sees = (at >= key) & ((at < key + window) if window else True)
        lost[b, sees, 4 * head: 4 * head + 4, 32 * group: 32 * group + 32] = True
    cache.k_scales[0, 0, past + 150, 1] = float("nan")
    lost[0, (at >= past + 150) & ((at < past + 150 + window) if window else True), :4] = True
    out = kv4_attend(q, cache, start, window=window)
    assert torch.equal(out.isnan(), lost)
    assert torch.equal(out.masked_fill(lost, 0), want.masked_fill(lost, 0))
    assert lib.ternaspmm_last_status() == 0


def test_infinite_and_nan_inputs_stay_in_their_group(lib):
    cache = KV4Cache.empty(1, 1, 64, 128)
    x = torch.ones((1, 1, 1, 128), device="cuda", dtype=torch.bfloat16)
    x[..., 3], x[..., 40], x[..., 70] = float("nan"), float("inf"), 3e38
    kv4_append(cache, x, x, torch.zeros(1, dtype=torch.int64, device="cuda"))
    k, v = kv4_read(cache, torch.zeros(1, dtype=torch.int64, device="cuda"), 1)
    for y in (k, v):
        assert y[..., :32].isnan().all() and not y[..., 32:64].isfinite().any() and not y[..., 64:96].isfinite().any() and y[..., 96:].eq(1).all()


def test_sequences_outside_of_the_cache(lib):
    cache, k, v = filled(4, 1, 64, 64, 6)
    before = [t.clone() for t in (cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales)]
    x = torch.ones((4, 3, 1, 64), device="cuda", dtype=torch.bfloat16)
    table = rotary_table(64, 64)
    for start, counts in (([-1, 62, 2 ** 40, -2 ** 62], None), ([0, 0, 63, 2 ** 63 - 1], [4, -1, 2, 3])):
        start, counts = torch.tensor(start, device="cuda"), None if counts is None else torch.tensor(counts, device="cuda")
        kv4_append(cache, x, x, start, counts, q=x, table=table)
        assert lib.ternaspmm_last_status() == 1
        assert all(torch.equal(a, b) for a, b in zip(before, (cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales)))
        assert kv4_attend(x, cache, start, counts).isnan().all() and lib.ternaspmm_last_status() == 1
        assert all(t.isnan().all() for t in kv4_read(cache, start, 3, counts)) and lib.ternaspmm_last_status() == 1
    # one of them among others
    start = torch.tensor([5, 61, 62, 0], device="cuda")
    out = kv4_attend(x, cache, start)
    assert out.isnan().flatten(1).all(1).tolist() == [False, False, True, False] and lib.ternaspmm_last_status() == 1
    ref, tol = attention(x, k, v, start, torch.full_like(start, 3), 0, 0.125)
    assert ((out.double() - ref).abs() <= tol)[[0, 1, 3]].all()
    assert lib.ternaspmm_last_status() == 0


def test_two_graphs_and_streams(lib):
    """Captured calls keep their workspaces apart, replay on new lengths, and run beside each other."""
    B, H, K, D, L = 2, 8, 2, 128, 4096
    cache, k, v = filled(B, K, L, D, 7)
    q = [torch.randn((B, 1, H, D), generator=gen(i), device="cuda").to(torch.bfloat16) for i in range(2)]
    start = [torch.tensor([900, 4000], device="cuda"), torch.tensor([4095, 17], device="cuda")]
    kv4_attend(q[0], cache, start[0])
    graphs, outs, streams = [torch.cuda.CUDAGraph() for _ in q], [], [torch.cuda.Stream() for _ in q]
    for g, x, s in zip(graphs, q, start):
        with torch.cuda.graph(g):
            outs.append(kv4_attend(x, cache, s))
    for s in start:
        s.copy_(torch.randint(0, L, (B,), device="cuda"))
    torch.cuda.synchronize()
    for _ in range(20):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for o, x, s in zip(outs, q, start):
        assert torch.equal(o, check(x, cache, k, v, s))


def test_two_graphs_of_many_tokens(lib):
    """The same with the keys in parts, whose results meet in a workspace."""
    B, T, H, K, D, L = 2, 80, 8, 2, 128, 2048
    cache, k, v = filled(B, K, L, D, 7)
    q = [torch.randn((B, T, H, D), generator=gen(i), device="cuda").to(torch.bfloat16) for i in range(2)]
    start = [torch.tensor([900, 1700], device="cuda"), torch.tensor([L - T, 17], device="cuda")]
    kv4_attend(q[0], cache, start[0])
    graphs, outs, streams = [torch.cuda.CUDAGraph() for _ in q], [], [torch.cuda.Stream() for _ in q]
    for g, x, s in zip(graphs, q, start):
        with torch.cuda.graph(g):
            outs.append(kv4_attend(x, cache, s))
    for s in start:
        s.copy_(torch.randint(0, L - T, (B,), device="cuda"))
    torch.cuda.synchronize()
    for _ in range(20):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for o, x, s in zip(outs, q, start):
        assert torch.equal(o, check(x, cache, k, v, s))


def test_offsets_beyond_32_bits(lib):
    """A cache of 6 GB a side: the last tokens of the last sequence, through every entry."""
    B, H, K, D, L = 40, 16, 8, 128, 262144
    big = KV4Cache.empty(B, K, L, D)
    assert big.k_codes.numel() > 1 << 32
    g = gen(20)
    k, v = (torch.randn((1, 128, K, D), generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    at = torch.full((B,), L - 128, device="cuda")
    counts = torch.zeros(B, dtype=torch.int64, device="cuda")
    counts[-1] = 128
    kv4_append(big, k.expand(B, -1, -1, -1), v.expand(B, -1, -1, -1), at, counts)
    got_k, got_v = kv4_read(big, at, 128, counts)
    lk, lv = levels(k)[0], levels(v)[0]
    assert torch.equal(got_k[-1:], lk.to(torch.bfloat16)) and torch.equal(got_v[-1:], lv.to(torch.bfloat16)) and not got_k[:-1].any()
    for T in (1, 3, 40):                  # (no other sequence has values there; a window keeps to what was written)
        q = torch.randn((B, T, H, D), generator=g, device="cuda").to(torch.bfloat16)
        out = kv4_attend(q, big, torch.full((B,), L - T, device="cuda"), window=60)
        want, tol = attention(q[-1:], lk, lv, torch.tensor([128 - T], device="cuda"), torch.tensor([T], device="cuda"), 60, D ** -0.5)
        assert ((out[-1:].double() - want).abs() <= tol).all() and not out[:-1].any()
    assert lib.ternaspmm_last_status() == 0


def test_refusals(lib):
    cache = KV4Cache.empty(2, 2, 64, 64)
    x, start = torch.zeros((2, 3, 2, 64), device="cuda", dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int64, device="cuda")
    table = rotary_table(64, 64)
    for bad in (dict(k=x.float()), dict(v=x[:, :2]), dict(k=x[:1]), dict(k=x[:, :, :1]), dict(k=x[..., :32]), dict(start=start.int()), dict(start=start[:0]),
                dict(counts=start[:1]), dict(q=x), dict(table=rotary_table(128, 64)), dict(q=x[:, :2], table=table), dict(k=x.cpu())):
        with pytest.raises((ValueError, RuntimeError)):
            kv4_append(**{**dict(cache=cache, k=x, v=x, start=start), **bad})
    for bad in (dict(q=x[:, :, :1]), dict(q=x.half()), dict(window=-1), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(start=start.cpu())):
        with pytest.raises((ValueError, RuntimeError)):
            kv4_attend(**{**dict(q=x, cache=cache, start=start), **bad})
    for bad in (dict(max_len=0), dict(head_dim=96), dict(batch=0)):
        with pytest.raises(ValueError):
            KV4Cache.empty(**{**dict(batch=1, kv_heads=1, max_len=64, head_dim=64), **bad})
    leaf = x.clone().requires_grad_()
    for call in (lambda: kv4_append(cache, leaf, x, start), lambda: kv4_attend(leaf, cache, start)):
        with pytest.raises(RuntimeError, match="gradient"):
            call()
    with torch.no_grad():
        kv4_attend(leaf, cache, start)
    with pytest.raises(ValueError):
        KV4Cache(cache.k_codes[:, :, :60].contiguous(), *(t[:, :, :60].contiguous() for t in (cache.k_scales, cache.v_codes, cache.v_scales)))
    assert kv4_attend(x[:, :0], cache, start).shape == (2, 0, 2, 64) and kv4_append(cache, x[:, :0], x[:, :0], start) is None
    assert lib.ternaspmm_last_status() == 0
