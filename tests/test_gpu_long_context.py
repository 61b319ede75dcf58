"""GPU: rotation, 4-bit cache, attention over it and scores as they are used together - a prompt, then token by token, in the model
and in the generation loop."""
import math

import pytest
import torch

from test_gpu_kv4 import attention, levels
from ternainfer_b200 import model as model_module
from ternainfer_b200.convert.convert_TernaInfer import random_checkpoint
from ternainfer_b200.generate import FastGen, GenArgs
from ternainfer_b200.kv4 import KV4Cache, kv4_append, kv4_attend, kv4_read
from ternainfer_b200.model import ModelArgs, Transformer
from ternainfer_b200.rotary import rotary_table, rotate
from ternainfer_b200.scores import token_logprobs

pytestmark = pytest.mark.gpu


def build(max_len=160, layers=2, vocab=1024, **kw):
    args = ModelArgs(n_layers=layers, vocab_size=vocab, **kw)
    dic = random_checkpoint(args.dim, layers, args.n_heads, args.n_kv_heads, args.ffn_dim, vocab, seed=11)
    for key in dic:                 # sub-layers that change the residual stream by about a per cent, as a trained network's do
        if key.endswith(("wo.weight_scale", "w2.weight_scale")):
            dic[key] = dic[key] * 2.5e-4
    with torch.device("cuda"):
        return Transformer(args, dic, max_seq_len=max_len).to(torch.bfloat16)


@pytest.mark.parametrize("D,H,K", [(128, 20, 5), (64, 12, 4)])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_prompt_then_tokens(lib, D, H, K, layout):
    """Sequences of different lengths in a padded prompt, then one token each at a time: every result against float64."""
    B, T, L = 3, 23, 64
    g = torch.Generator(device="cuda").manual_seed(D)
    table = rotary_table(D, L, layout=layout, rotary_dim=D // 2, scaling=dict(type="yarn", factor=4, original_len=16))
    cache = KV4Cache.empty(B, K, L, D)
    k_all, v_all = (torch.zeros((B, L, K, D), dtype=torch.float64, device="cuda") for _ in range(2))
    start, counts = torch.zeros(B, dtype=torch.int64, device="cuda"), torch.tensor([23, 7, 16], device="cuda")
    for step in range(8):
        n = T if step == 0 else 1
        q, k, v = torch.randn((B, n, H + 2 * K, D), generator=g, device="cuda").to(torch.bfloat16).split([H, K, K], 2)
        c = counts if step == 0 else torch.ones_like(counts)
        pos = start[:, None] + torch.arange(n, device="cuda")
        want_q, want_k = rotate(q, k, table, pos)
        got_q = kv4_append(cache, k, v, start, c if step == 0 else None, q=q, table=table)
        assert torch.equal(got_q, want_q)
        for b in range(B):
            at = slice(int(start[b]), int(start[b] + c[b]))
            k_all[b, at], v_all[b, at] = levels(want_k)[0][b, :c[b]], levels(v)[0][b, :c[b]]
        out = kv4_attend(got_q, cache, start, c if step == 0 else None)
        want, tol = attention(want_q, k_all, v_all, start, c, 0, D ** -0.5)
        assert ((out.double() - want).abs() <= tol).all()
        start = start + c
    assert lib.ternaspmm_last_status() == 0


@torch.inference_mode()
@pytest.mark.parametrize("fused", [False, True])
def test_model_with_a_4_bit_cache(lib, fused, monkeypatch):
    """The model on the kernels against the same model on plain operators, a prompt and a token; both round the same values to bf16
    and differ in single roundings of attention results."""
    m = build(kv_bits=4, fused_glue=fused)
    g = torch.Generator(device="cuda").manual_seed(5)
    tok = torch.randint(0, 1024, (2, 75), generator=g, device="cuda")
    nxt = torch.randint(0, 1024, (2, 1), generator=g, device="cuda")
    cache = m.make_cache(2, "cuda")
    assert isinstance(cache[0], KV4Cache)
    got = m(tok, cache, torch.arange(75, device="cuda")), m(nxt, cache, torch.tensor([75], device="cuda"))

    held = {}

    def append(c, k, v, start, counts=None, q=None, table=None):
        q, k = rotate(q, k, table, start + torch.arange(k.shape[1], device="cuda"))
        kk, vv = held.setdefault(id(c), tuple(torch.zeros((2, c.max_len, 5, 128), dtype=torch.float64, device="cuda") for _ in range(2)))
        kk[:, int(start): int(start) + k.shape[1]], vv[:, int(start): int(start) + k.shape[1]] = levels(k)[0], levels(v)[0]
        return q

    def attend(q, c, start):
        return attention(q, *held[id(c)], start.expand(2), torch.full((2,), q.shape[1], device="cuda"), 0, 128 ** -0.5)[0].to(torch.bfloat16)

    monkeypatch.setattr(model_module, "kv4_append", append)
    monkeypatch.setattr(model_module, "kv4_attend", attend)
    cache = m.make_cache(2, "cuda")
    want = m(tok, cache, torch.arange(75, device="cuda")), m(nxt, cache, torch.tensor([75], device="cuda"))
    for a, b in zip(got, want):
        # Logits are bf16: eight significant bits, so neighbours between 2^e and 2^(e+1) are 2^(e-7) apart, up to 2^-7 of the value, and two that
        # are rounded alike up to a last place differ by one such step.  On average: two roundings of up to half a step, 2^-8,
        # evenly spread, sqrt(2 / 3) * 2^-8 together.
        assert (a - b).abs().max() <= 2.0 ** -7 * b.abs().max() and ((a - b).norm() / b.norm()) < 2.0 ** -8
    assert lib.ternaspmm_last_status() == 0


@torch.inference_mode()
@pytest.mark.parametrize("fused", [False, True])
def test_layouts_of_the_model(lib, fused):
    """Half layout on rows put in its order is the interleaved model: the attention's sums alone are taken in another order."""
    perm = torch.cat([torch.arange(0, 128, 2), torch.arange(1, 128, 2)]).cuda()
    for kw in (dict(kv_bits=16), dict(kv_bits=16, rope_scaling=dict(type="linear", factor=3.0))):
        a, b = build(fused_glue=fused, flash_attention=False, **kw), build(fused_glue=fused, rope_layout="half", **kw)
        for x, y in zip(a.layers, b.layers):
            wqkv = y.attention.wqkv

            def reordered(out):
                q, k, v = out.split([2560, 640, 640], -1)
                return torch.cat([q.unflatten(-1, (-1, 128))[..., perm].flatten(-2), k.unflatten(-1, (-1, 128))[..., perm].flatten(-2), v], -1)
            y.attention.wqkv = type("W", (torch.nn.Module,), dict(
                forward=lambda self, x, w=wqkv: reordered(w(x)), forward_normed=lambda self, x, n, e, w=wqkv: reordered(w.forward_normed(x, n, e))))()
        g = torch.Generator(device="cuda").manual_seed(3)
        tok = torch.randint(0, 1024, (2, 33), generator=g, device="cuda")
        ca, cb = a.make_cache(2, "cuda"), b.make_cache(2, "cuda")
        for t, pos in ((tok, torch.arange(33, device="cuda")), (tok[:, :1], torch.tensor([33], device="cuda"))):
            x, y = a(t, ca, pos), b(t, cb, pos)
            assert (x - y).abs().max() <= 2.0 ** -7 * x.abs().max() and (x - y).norm() / x.norm() < 2.0 ** -8


@torch.inference_mode()
def test_generation_loop(lib):
    """Graphs over a 4-bit cache give the eager loop's tokens, and score() the log probabilities of the logits that forward() gives."""
    m = build(kv_bits=4, fused_glue=True, rope_layout="half", rotary_dim=64)
    prompt = torch.randint(0, 1024, (2, 40), generator=torch.Generator(device="cuda").manual_seed(2), device="cuda")
    gen = FastGen(m, GenArgs(12, 2, 40, True))
    a, _ = gen.generate(prompt)
    b, _ = FastGen(m, GenArgs(12, 2, 40, False)).generate(prompt)
    assert torch.equal(a, b)
    tokens = torch.cat([prompt, a], 1)
    r = m.score(tokens, gen.cache, top=3)
    logits = m(tokens[:, :-1], m.make_cache(2, "cuda"), torch.arange(51, device="cuda"))
    want = token_logprobs(logits, tokens[:, 1:], 3)
    assert r.logprob.shape == (2, 51) and r.top_token.shape == (2, 51, 3)
    # (bf16 logits in one, the same values as fp32 in the other: threads add them up in another order, fp32 sums of 1024 terms)
    assert torch.equal(r.top_token, want.top_token) and all((x - y).abs().max() <= 1e-5 for x, y in zip(r[:3], want[:3]))
    exact = torch.log_softmax(logits.double(), -1).gather(-1, tokens[:, 1:, None])[..., 0]
    assert ((r.logprob.double() - exact).abs() <= 1e-5).all()
    with pytest.raises(ValueError):
        m.score(tokens[:, :1])
    for bad in (dict(kv_bits=8), dict(rope_layout="other"), dict(kv_bits=4, n_heads=40, n_kv_heads=10, dim=1280)):
        with pytest.raises(ValueError):
            Transformer(ModelArgs(n_layers=0, **bad), dict(**{"tok_embeddings.weight": torch.zeros((128256, bad.get("dim", 2560))), "norm.weight": torch.zeros(bad.get("dim", 2560))}))


def test_command(lib, capsys, monkeypatch):
    import sys
    from ternainfer_b200 import generate
    monkeypatch.setattr(sys, "argv", "generate --layers 1 --prompt_length 20 --gen_length 5 --kv_bits 4 --rope_layout half --rope_linear 4 --top_logprobs 2 --fused_glue".split())
    generate.main()
    assert "log probability per generated token -" in capsys.readouterr().out


def test_empty_calls(lib):
    """No rows, no tokens, no sequences; a single row without leading dimensions; transposed, sliced and broadcast logits."""
    for lead in ((0,), (2, 0), ()):
        x, t = torch.randn(*lead, 50, device="cuda", requires_grad=True), torch.zeros(lead, dtype=torch.int64, device="cuda")
        r = token_logprobs(x, t, 3)
        assert r.logprob.shape == lead and r.top_token.shape == (*lead, 3)
        assert torch.autograd.grad(r.logprob.sum() + r.entropy.sum(), x)[0].shape == x.shape
    cache, start = KV4Cache.empty(2, 2, 64, 64), torch.zeros(2, dtype=torch.int64, device="cuda")
    none = torch.randn(2, 0, 2, 64, device="cuda").bfloat16()
    assert kv4_append(cache, none, none, start) is None and kv4_attend(none, cache, start).shape == none.shape
    assert all(t.shape == none.shape for t in kv4_read(cache, start, 0))
    for shape in ((0, 3, 2, 64), (2, 0, 2, 64)):
        q = torch.randn(shape, device="cuda", requires_grad=True)
        a, b = rotate(q, q.detach(), rotary_table(64, 64), torch.zeros(shape[1], dtype=torch.int64, device="cuda"))
        assert a.shape == b.shape == torch.autograd.grad(a.sum(), q)[0].shape == shape
    t = torch.zeros(8, dtype=torch.int64, device="cuda")
    for x in (torch.randn(50, 8, device="cuda").t(), torch.randn(8, 101, device="cuda")[:, 1:51], torch.randn(50, device="cuda").expand(8, 50)):
        x.requires_grad_()
        y = token_logprobs(x, t)
        want = torch.log_softmax(x.double(), -1)[:, 0]
        assert ((y.logprob.double() - want).abs() <= 2.0 ** -19 + want.abs() * 2.0 ** -22).all()
        assert torch.autograd.grad(y.logprob.sum(), x)[0].shape == x.shape
    assert lib.ternaspmm_last_status() == 0


FAILED_LAUNCH = """
import torch
from ternainfer_b200.kv4 import KV4Cache, kv4_append, kv4_attend, kv4_read
from ternainfer_b200.rotary import rotary_table, rotate
from ternainfer_b200.scores import token_logprobs
x = torch.randn((1, 2, 4, 64), device="cuda").bfloat16()
table, pos, start = rotary_table(64, 64), torch.arange(2, device="cuda"), torch.zeros(1, dtype=torch.int64, device="cuda")
cache = KV4Cache.empty(1, 4, 64, 64)
logits, targets = torch.randn((2, 50), device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda")
calls = (lambda: rotate(x, x, table, pos), lambda: kv4_append(cache, x, x, start, q=x, table=table), lambda: kv4_read(cache, start, 2),
         lambda: kv4_attend(x, cache, start), lambda: token_logprobs(logits, targets, 3))
want = [f() for f in calls]
torch.cuda.synchronize()
stream = torch.cuda.Stream()
try:
    with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=stream):
        try:
            stream.synchronize()                # not allowed: nothing can be launched into this capture any more
        except RuntimeError:
            pass
        for f in calls:
            try:
                f()
            except RuntimeError:
                print("refused")
except RuntimeError:
    print("capture over")
torch.cuda.synchronize()
flat = lambda r: [t for t in (r if isinstance(r, tuple) else (r,)) if t is not None]
print("the same", all(torch.equal(a, b) for f, w in zip(calls, want) for a, b in zip(flat(f()), flat(w))))
"""


def test_a_launch_that_fails_is_an_error_of_the_call():
    import subprocess
    import sys
    from pathlib import Path
    r = subprocess.run([sys.executable, "-c", FAILED_LAUNCH], capture_output=True, text=True, timeout=300, cwd=Path(__file__).resolve().parents[1])
    assert r.returncode == 0 and r.stdout.split("\n")[:7] == ["refused"] * 5 + ["capture over", "the same True"], r.stdout + r.stderr


CAPTURED_GRADIENT = """
import sys
import torch
from ternainfer_b200.rotary import rotary_table, rotate
from ternainfer_b200.scores import token_logprobs
table, pos, t = rotary_table(64, 64), torch.arange(8, device="cuda"), torch.zeros(8, dtype=torch.int64, device="cuda")
for shape, call in (((1, 8, 4, 64), lambda x: rotate(x, None, table, pos)[0]), ((8, 500), lambda x: token_logprobs(x, t)[0])):
    x = torch.randn(shape, device="cuda", requires_grad=True)
    w = torch.randn_like(call(x))
    want, = torch.autograd.grad(call(x), x, w)
    x.grad = torch.zeros_like(x)
    torch.cuda.synchronize()
    kept = call(x) if sys.argv[1] == "kept" else None
    g = torch.cuda.CUDAGraph()
    try:
        with torch.cuda.graph(g):
            call(x).backward(w)
        x.grad.zero_()
        g.replay()
        torch.cuda.synchronize()
        print("replayed", torch.equal(x.grad, want))
    except RuntimeError:
        print("refused")
    if kept is not None:
        x.grad = None
        kept.backward(w)
        print("eager", torch.equal(x.grad, want))
        break
"""


@pytest.mark.parametrize("which,said", [("none", ["replayed True", "replayed True"]), ("kept", ["refused", "eager True"])])
def test_captured_gradients(which, said):
    """A backward pass in a graph; with an eager graph of the same leaf alive torch lets none be captured, which ends neither the process nor that one."""
    import subprocess
    import sys
    from pathlib import Path
    r = subprocess.run([sys.executable, "-c", CAPTURED_GRADIENT, which], capture_output=True, text=True, timeout=300, cwd=Path(__file__).resolve().parents[1])
    assert r.returncode == 0 and r.stdout.split("\n")[:-1] == said, r.stdout + r.stderr
