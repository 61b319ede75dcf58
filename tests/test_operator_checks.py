"""CPU: what the rotary, 4-bit cache and scoring operators refuse before anything is launched, and the frequencies of scaled rotations."""
import ctypes
import math

import pytest
import torch

from ternainfer_b200.kv4 import KV4Cache, kv4_append, kv4_attend, kv4_read
from ternainfer_b200.rotary import RotaryTable, rotary_frequencies, rotary_table, rotate
from ternainfer_b200.scores import token_logprobs

P = 1 << 20                     # an aligned address that nothing reads: every call below is refused on the host


def strides(*v):
    return (ctypes.c_longlong * 3)(*v)


def test_cpu_tensors_are_refused():
    x, pos = torch.zeros((1, 2, 1, 64), dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int64)
    table, cache = rotary_table(64, 8, device="cpu"), KV4Cache.empty(1, 1, 64, 64, device="cpu")
    for call in (lambda: rotate(x, None, table, pos), lambda: kv4_append(cache, x, x, pos[:1]), lambda: kv4_read(cache, pos[:1], 2),
                 lambda: kv4_attend(x, cache, pos[:1]), lambda: token_logprobs(torch.zeros((2, 5)), pos)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()
    with pytest.raises(ValueError, match="-12 tokens"):      # (a message with a number: the extension and torch share one libstdc++)
        kv4_read(cache, pos[:1], -12)


def test_cache_shapes():
    c = KV4Cache.empty(2, 3, 100, 128, device="cpu")
    assert (c.batch, c.kv_heads, c.max_len, c.head_dim) == (2, 3, 128, 128)
    assert c.k_codes.shape == (2, 3, 128, 64) and c.v_scales.shape == (2, 3, 128, 4)
    for bad in ((c.k_codes.float(), c.k_scales, c.v_codes, c.v_scales), (c.k_codes, c.k_scales[..., :2], c.v_codes, c.v_scales),
                (c.k_codes, c.k_scales, c.v_codes.transpose(1, 2), c.v_scales)):
        with pytest.raises(ValueError):
            KV4Cache(*bad)


def test_frequencies():
    theta, n = 10000.0, 32
    plain, one = rotary_frequencies(n, theta)
    assert one == 1 and torch.equal(plain, theta ** (-torch.arange(0, n, 2, dtype=torch.float64) / n))
    assert torch.equal(rotary_frequencies(n, theta, dict(type="linear", factor=3))[0], plain / 3)
    ntk = rotary_frequencies(n, theta, dict(type="ntk", factor=3))[0]
    assert ntk[0] == plain[0] and abs(ntk[-1] * 3 / plain[-1] - 1) < 1e-12
    for scaling in (dict(type="yarn", factor=5, original_len=4096), dict(type="wavelength", factor=5, original_len=4096)):
        inv, size = rotary_frequencies(n, theta, scaling)
        turns = 4096 * plain / (2 * math.pi)
        ratio = plain / inv
        assert (ratio[turns > 32] == 1).all() and (abs(ratio[turns < 1] - 5) < 1e-12).all() and (ratio[1:] >= ratio[:-1]).all() and 1 < ratio[(turns > 3) & (turns < 4)].min()
        assert size == (0.1 * math.log(5) + 1 if scaling["type"] == "yarn" else 1)
    for bad in (dict(type="other", factor=2), dict(type="linear"), dict(type="linear", factor=-1), dict(type="linear", factor=2, low=3), dict(type="yarn", factor=2),
                dict(type="wavelength", factor=2, original_len=9, low=4, high=4)):
        with pytest.raises(ValueError):
            rotary_frequencies(n, theta, bad)
    for bad in (0, 1, 7):
        with pytest.raises(ValueError):
            rotary_frequencies(bad)
    with pytest.raises(ValueError):
        rotary_table(64, 8, rotary_dim=128, device="cpu")
    with pytest.raises(ValueError):
        RotaryTable(torch.zeros(3, 4), torch.zeros(3, 4), "other")


def test_rotate_statuses(lib):
    good = dict(q=P, qs=strides(64, 64, 64), qh=1, qo=P, k=None, ks=None, kh=0, ko=None, type=0, cos=P, sin=P, len=4, rot=64, half=0, inv=0, pos=P, sb=0, st=1,
                batch=1, tokens=1, dim=64)
    for status, change in ((1, dict(batch=0)), (1, dict(tokens=0)), (1, dict(qh=0)), (1, dict(kh=-1)), (1, dict(dim=63)), (1, dict(rot=66)), (1, dict(rot=7)),
                           (1, dict(len=0)), (1, dict(type=3)), (2, dict(q=None)), (2, dict(qo=None)), (2, dict(kh=1)), (2, dict(cos=None)), (2, dict(pos=None)),
                           (2, dict(q=P + 1)), (2, dict(qs=None))):
        assert lib.ternaspmm_rotate(*{**good, **change}.values(), None) == status, change
        assert lib.ternaspmm_last_status() == status


def test_kv4_statuses(lib):
    s = strides(64, 64, 64)
    append = dict(kc=P, ks=P, vc=P, vs=P, L=64, k=P, kst=s, v=P, vst=s, q=None, qst=None, qo=None, cos=None, sin=None, len=0, rot=0, half=0, start=P, ss=1, counts=None,
                  batch=1, tokens=1, heads=0, kv=1, dim=64)
    for status, change in ((1, dict(batch=0)), (1, dict(batch=65536)), (1, dict(tokens=0)), (1, dict(kv=0)), (1, dict(dim=96)), (1, dict(L=0)), (1, dict(L=100)),
                           (1, dict(cos=P, sin=P, rot=66, len=4)), (1, dict(q=P, heads=0)), (2, dict(kc=None)), (2, dict(vs=P + 8)), (2, dict(k=None)),
                           (2, dict(k=P + 2)), (2, dict(vst=strides(64, 64, 2))), (2, dict(start=None)), (2, dict(cos=P, rot=64, len=4)),
                           (2, dict(q=P, qst=s, qo=P, heads=1)), (2, dict(q=P, qst=s, heads=1, cos=P, sin=P, rot=64, len=4))):
        assert lib.ternaspmm_kv4_append(*{**append, **change}.values(), None) == status, change
    read = dict(kc=P, ks=P, vc=P, vs=P, L=64, start=P, ss=1, counts=None, k=P, v=P, batch=1, tokens=1, kv=1, dim=64)
    for status, change in ((1, dict(L=96)), (1, dict(tokens=-1)), (2, dict(k=None)), (2, dict(v=P + 4)), (2, dict(start=None))):
        assert lib.ternaspmm_kv4_read(*{**read, **change}.values(), None) == status, change
    attend = dict(q=P, qst=s, kc=P, ks=P, vc=P, vs=P, L=64, start=P, ss=1, counts=None, window=0, scale=0.125, out=P, batch=1, tokens=1, heads=2, kv=1, dim=64, ws=P,
                  bytes=1 << 40)
    for status, change in ((1, dict(heads=3, kv=2)), (1, dict(heads=0)), (1, dict(window=-1)), (1, dict(scale=0.0)), (1, dict(scale=math.nan)), (1, dict(scale=math.inf)),
                           (1, dict(bytes=-1)), (1, dict(dim=32)), (1, dict(tokens=1 << 30)), (2, dict(q=P + 8)), (2, dict(qst=strides(64, 64, 4))), (2, dict(out=None)),
                           (2, dict(ks=None))):
        assert lib.ternaspmm_kv4_attend(*{**attend, **change}.values(), None) == status, change
    assert lib.ternaspmm_kv4_attend_workspace(1, 1, 3, 2, 64, 64) == -1 and lib.ternaspmm_kv4_attend_workspace(1, 1, 4, 2, 64, 1 << 20) >= 0


def test_logprob_statuses(lib):
    good = dict(x=P, ld=10, type=0, t=P, rows=1, vocab=10, top=2, lp=P, h=P, lse=P, tl=P, tt=P, ws=P, bytes=1 << 30)
    for status, change in ((1, dict(rows=0)), (1, dict(vocab=0)), (1, dict(ld=9)), (1, dict(type=-1)), (1, dict(top=33, vocab=50, ld=50)), (1, dict(top=11)), (1, dict(top=-1)),
                           (1, dict(vocab=(1 << 19) + 1, ld=1 << 21)),
                           (1, dict(bytes=15)), (1, dict(vocab=20000, ld=20000, bytes=287)), (2, dict(x=None)), (2, dict(x=P + 1)), (2, dict(t=None)), (2, dict(lse=None)), (2, dict(tt=None)), (2, dict(ws=None)),
                           (2, dict(ws=P + 8))):
        assert lib.ternaspmm_token_logprobs(*{**good, **change}.values(), None) == status, change
    # short rows need next to nothing, longer ones the sums of eight warps and two alternatives for each 32 KB
    assert lib.ternaspmm_token_logprobs_workspace(1, 10, 0, 2) == 16 and lib.ternaspmm_token_logprobs_workspace(1, 20000, 0, 2) == 288
    assert lib.ternaspmm_token_logprobs_workspace(1, 10, 0, 11) == -1
    grad = dict(x=P, ld=10, type=2, t=P, rows=1, vocab=10, lse=P, h=P, gl=None, gh=P, out=P)
    for status, change in ((1, dict(rows=0)), (1, dict(ld=9)), (2, dict(out=P + 2)), (2, dict(h=None))):
        assert lib.ternaspmm_token_logprobs_grad(*{**grad, **change}.values(), None) == status, change


def test_forward_mode_is_refused():
    """A tensor with a tangent but no gradient of its own: an error, not a result whose tangent counts as zero."""
    import torch.autograd.forward_ad as forward_ad
    x, pos = torch.zeros((1, 2, 1, 64), dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int64)
    table, cache = rotary_table(64, 8, device="cpu"), KV4Cache.empty(1, 1, 64, 64, device="cpu")
    with forward_ad.dual_level():
        d = forward_ad.make_dual(x, torch.ones_like(x))
        cos = forward_ad.make_dual(table.cos, torch.ones_like(table.cos))
        logits = forward_ad.make_dual(torch.zeros((2, 5)), torch.ones((2, 5)))
        for call in (lambda: rotate(d, None, table, pos), lambda: rotate(x, d, table, pos), lambda: rotate(x, None, RotaryTable(cos, table.sin), pos),
                     lambda: kv4_append(cache, d, x, pos[:1]), lambda: kv4_append(cache, x, d, pos[:1]), lambda: kv4_append(cache, x, x, pos[:1], q=d, table=table),
                     lambda: kv4_attend(d, cache, pos[:1]), lambda: token_logprobs(logits, pos)):
            with pytest.raises(NotImplementedError, match="tangent"):
                call()
        with pytest.raises(RuntimeError, match="no CPU path"):            # (as before without one)
            token_logprobs(forward_ad.unpack_dual(logits).primal, pos)


def test_sizes_that_no_launch_takes(lib):
    rotate_args = dict(q=P, qs=strides(6, 6, 6), qh=2, qo=P, k=None, ks=None, kh=0, ko=None, type=0, cos=P, sin=P, len=4, rot=2, half=1, inv=0, pos=P, sb=0, st=1,
                       batch=1, tokens=1 << 30, dim=6)
    assert lib.ternaspmm_rotate(*rotate_args.values(), None) == 1 and lib.ternaspmm_last_status() == 1
    with pytest.raises(ValueError, match="65536"):
        KV4Cache.empty(65536, 1, 64, 64, device="meta")
    assert KV4Cache.empty(65535, 1, 64, 64, device="meta").batch == 65535


def test_logprob_rows(lib):
    many = (1 << 23) + 1
    assert lib.ternaspmm_token_logprobs_workspace(many, 1 << 14, 0, 0) == 16 == lib.ternaspmm_token_logprobs_workspace((1 << 31) - 1, 1 << 13, 2, 0)
    assert lib.ternaspmm_token_logprobs_workspace(many, (1 << 14) + 1, 0, 0) == -1 == lib.ternaspmm_token_logprobs_workspace(1, (1 << 31) - 1, 0, 0)


def test_gradients_of_tables_and_caches_are_refused():
    x, pos = torch.zeros((1, 2, 1, 64), dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int64)
    plain, c = rotary_table(64, 8, device="cpu"), KV4Cache.empty(1, 1, 64, 64, device="cpu")
    leaf = lambda t: t.clone().requires_grad_()
    for table in (RotaryTable(leaf(plain.cos), plain.sin), RotaryTable(plain.cos, leaf(plain.sin))):
        for call in (lambda: rotate(x, None, table, pos), lambda: kv4_append(c, x, x, pos[:1], table=table)):
            with pytest.raises(RuntimeError, match="requires a gradient"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU path"):
                call()
    for cache in (KV4Cache(c.k_codes, leaf(c.k_scales), c.v_codes, c.v_scales), KV4Cache(c.k_codes, c.k_scales, c.v_codes, leaf(c.v_scales))):
        for call in (lambda: kv4_append(cache, x, x, pos[:1]), lambda: kv4_read(cache, pos[:1], 2), lambda: kv4_attend(x, cache, pos[:1])):
            with pytest.raises(RuntimeError, match="requires a gradient"):
                call()


def test_frequencies_that_do_not_exist():
    """Wrong numbers are ValueErrors: no table of NaN, and no division by zero on the way."""
    for theta in (-10000.0, 0.0, math.nan):
        with pytest.raises(ValueError, match="theta"):
            rotary_frequencies(32, theta)
    yarn = dict(type="yarn", factor=4, original_len=4096)
    for theta, scaling in ((1.0, yarn), (10000.0, dict(yarn, beta_fast=0)), (10000.0, dict(yarn, beta_slow=0)), (10000.0, dict(yarn, beta_slow=-1)),
                           (10000.0, dict(yarn, beta_fast=1, beta_slow=32)), (10000.0, dict(yarn, original_len=0)),
                           (10000.0, dict(type="wavelength", factor=4, original_len=-4096))):
        with pytest.raises(ValueError, match="yarn|original_len"):
            rotary_frequencies(32, theta, scaling)
    assert torch.equal(rotary_frequencies(32, 1.0)[0], torch.ones(16, dtype=torch.float64))
