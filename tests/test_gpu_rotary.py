"""GPU: rotary positions against complex numbers in 64 bits, their gradient, tables, strides and refusals."""
import pytest
import torch

from ternainfer_b200.rotary import RotaryTable, rotary_table, rotate

pytestmark = pytest.mark.gpu
SCALINGS = [None, dict(type="linear", factor=4), dict(type="ntk", factor=4), dict(type="yarn", factor=16, original_len=512),
            dict(type="wavelength", factor=8, original_len=512)]


def turned(x, table, pos, back=False):
    """x [B, T, H, D] in float64: pairs as complex numbers times cos + i sin of the table; and a bound of what fp32 loses."""
    n = table.rotary_dim
    p = pos.expand(x.shape[:2])
    w = torch.complex(table.cos.double()[p], (-1 if back else 1) * table.sin.double()[p])[:, :, None]
    a, b = (slice(0, n // 2), slice(n // 2, n)) if table.layout == "half" else (slice(0, n, 2), slice(1, n, 2))
    y, lost = x.double().clone(), torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    z = torch.complex(y[..., a].contiguous(), y[..., b].contiguous()) * w
    # two products and a sum in fp32: at most a half step (2^-24) of each product and of the sum
    size = (y[..., a].abs() + y[..., b].abs()) * w.abs()
    lost[..., a] = lost[..., b] = size * 2.0 ** -23
    y[..., a], y[..., b] = z.real, z.imag
    return y, lost


def close(got, want, lost):
    tol = lost + (want.abs() + lost) * torch.finfo(got.dtype).eps / 2 + torch.finfo(got.dtype).tiny * torch.finfo(got.dtype).eps
    assert ((got.double() - want).abs() <= tol).all(), ((got.double() - want).abs() - tol).max()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("B,T,H,K,D,n", [(1, 1, 1, 1, 64, 64), (8, 1, 20, 5, 128, 128), (3, 7, 4, 2, 128, 40), (2, 33, 3, 3, 80, 20), (2, 5, 5, 1, 96, 96),
                                         (1, 2, 9, 2, 2, 2), (2, 3, 2, 1, 70, 6)])
def test_rotate(lib, dtype, layout, B, T, H, K, D, n):
    g = torch.Generator(device="cuda").manual_seed(B * T + D)
    qkv = torch.randn((B, T, H + 2 * K, D), generator=g, device="cuda").to(dtype)
    table = rotary_table(D, 300, 10000.0, rotary_dim=n, layout=layout)
    pos = torch.randint(0, 300, (B, T), generator=g, device="cuda")
    q, k = qkv[:, :, :H], qkv[:, :, H: H + K]
    got = rotate(q, k, table, pos)
    for x, y in zip((q, k), got):
        assert y.dtype == dtype and y.is_contiguous()
        close(y, *turned(x, table, pos))
    alone, none = rotate(q, None, table, pos)
    assert none is None and torch.equal(alone, got[0])
    shared = rotate(q, k, table, pos[0])
    close(shared[1], *turned(k, table, pos[:1]))
    assert lib.ternaspmm_last_status() == 0


@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_rotate_any_strides(lib, layout):
    g = torch.Generator(device="cuda").manual_seed(1)
    table = rotary_table(64, 99, rotary_dim=32, layout=layout)
    base = torch.randn((3, 6, 5, 131), generator=g, device="cuda").to(torch.bfloat16)
    pos = torch.randint(0, 99, (5, 12), generator=g, device="cuda")[:, ::2][:3]
    for x in (base[..., 1:65], base[..., 2:66], base[..., ::2][..., :64], base.transpose(1, 2)[..., 3:67].transpose(1, 2),
              torch.randn((3, 5, 6, 64), generator=g, device="cuda").to(torch.bfloat16).transpose(1, 2), base[:, :, :1, :64].expand(3, 6, 5, 64)):
        close(rotate(x, None, table, pos)[0], *turned(x, table, pos))
    assert rotate(base[:, :0, :, :64], base[:, :0, :1, :64], table, pos[:, :0])[0].shape == (3, 0, 5, 64)


def test_matches_the_decoders_rope(lib):
    """Adjacent pairs of a whole head of 128: bit for bit what linear.rope gives."""
    from ternainfer_b200.linear import rope
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn((2, 9, 5, 128), generator=g, device="cuda").to(torch.bfloat16)
    table = rotary_table(128, 700, 500000.0)
    pos = torch.arange(600, 609, device="cuda")
    assert torch.equal(rotate(x, None, table, pos)[0], rope(x, table.cos[pos].expand(2, 9, 64), table.sin[pos].expand(2, 9, 64)))


@pytest.mark.parametrize("scaling", SCALINGS)
def test_tables(scaling):
    """Far positions in 64 bits; what each kind of scaling says about the fastest and the slowest pair."""
    n, theta, far = 64, 500000.0, 131071
    t = rotary_table(64, far + 1, theta, scaling=scaling)
    inv = theta ** (-torch.arange(0, n, 2, dtype=torch.float64) / n)
    c, s = t.cos[far].double().cpu(), t.sin[far].double().cpu()
    kind = scaling["type"] if scaling else None
    size = 1.0 if kind != "yarn" else 0.1 * torch.log(torch.tensor(16.0, dtype=torch.float64)).item() + 1
    want = {None: inv, "linear": inv / 4, "ntk": inv * 4 ** -(torch.arange(32, dtype=torch.float64) / 31)}.get(kind)
    if want is None:                                   # the ends of the ramp; the pairs between lie between
        want = torch.stack([inv, inv / scaling["factor"]])
        turns = 512 * inv / (2 * torch.pi)
        assert turns[0] > 32 and turns[-1] < 1
        for i in (0, -1):
            a = far * want[-i, i]
            assert abs(c[i] - size * a.cos()) < 2e-7 and abs(s[i] - size * a.sin()) < 2e-7
    else:
        # half a step of fp32, and of the angle in 64 bits
        assert (c - (far * want).cos()).abs().max() < 2.0 ** -24 + 1e-10 and (s - (far * want).sin()).abs().max() < 2.0 ** -24 + 1e-10
    assert ((t.cos.double() ** 2 + t.sin.double() ** 2).sqrt() - size).abs().max() < 3e-7


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_gradient(lib, dtype, layout):
    g = torch.Generator(device="cuda").manual_seed(3)
    table = rotary_table(48, 50, rotary_dim=32, layout=layout, scaling=SCALINGS[3])
    pos = torch.randint(0, 50, (2, 7), generator=g, device="cuda")
    qk = torch.randn((2, 7, 6, 48), generator=g, device="cuda").to(dtype)
    q, k = qk[:, :, :4].detach().requires_grad_(), qk[:, :, 4:].detach().requires_grad_()
    gq, gk = torch.randn(q.shape, generator=g, device="cuda").to(dtype), torch.randn(k.shape, generator=g, device="cuda").to(dtype)
    got = torch.autograd.grad(rotate(q, k, table, pos), (q, k), (gq, gk))
    for x, y in zip((gq, gk), got):
        close(y, *turned(x, table, pos, back=True))
    # one side alone, a frozen one, a gradient of broadcast strides
    assert torch.equal(torch.autograd.grad(rotate(q, k.detach(), table, pos)[0], q, gq)[0], got[0])
    assert torch.equal(torch.autograd.grad(rotate(q.detach(), k, table, pos)[1], k, gk)[0], got[1])
    assert torch.equal(torch.autograd.grad(rotate(q, k, table, pos)[1], k, gk)[0], got[1])
    one = torch.ones((), device="cuda", dtype=dtype).expand(q.shape)
    close(torch.autograd.grad(rotate(q, None, table, pos)[0].sum(), q)[0], *turned(one, table, pos, back=True))
    if dtype == torch.float32:                         # against differences: rotation is linear, so these are exact up to rounding
        with torch.no_grad():
            d = torch.randn(q.shape, generator=g, device="cuda")
            diff = (((rotate(q + d, None, table, pos)[0].double() - rotate(q - d, None, table, pos)[0].double()) / 2) * gq.double()).sum()
        assert abs(diff - (got[0].double() * d.double()).sum()) < 1e-3


def test_positions_outside_of_the_table(lib):
    table = rotary_table(64, 20)
    x = torch.ones((2, 3, 2, 64), device="cuda", dtype=torch.bfloat16)
    y, _ = rotate(x, None, table, torch.tensor([[0, 19, 20], [-1, 5, 2 ** 40]], device="cuda"))
    assert lib.ternaspmm_last_status() == 1
    nan = y.isnan().flatten(2)
    assert nan.all(-1).tolist() == [[False, False, True], [True, False, True]] and nan.any(-1).equal(nan.all(-1))
    assert lib.ternaspmm_last_status() == 0


def test_streams_and_graphs(lib):
    g = torch.Generator(device="cuda").manual_seed(4)
    table = rotary_table(128, 64)
    q, k = (torch.randn((2, 3, h, 128), generator=g, device="cuda").to(torch.bfloat16) for h in (8, 2))
    pos = torch.arange(3, device="cuda")
    want = rotate(q, k, table, pos)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = rotate(q, k, table, pos)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = rotate(q, k, table, pos)
    pos += 7
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(out, rotate(q, k, table, pos)))


def test_refusals(lib):
    table = rotary_table(64, 20)
    q, pos = torch.zeros((2, 3, 2, 64), device="cuda", dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int64, device="cuda")
    for bad in (dict(q=q.double()), dict(q=q[0]), dict(k=q.float()), dict(k=q[:, :2]), dict(positions=pos.int()), dict(positions=pos[:2]),
                dict(positions=pos.cpu()), dict(q=q[..., :32]), dict(q=q[..., :63])):
        with pytest.raises((ValueError, RuntimeError)):
            rotate(**{**dict(q=q, k=None, table=table, positions=pos), **bad})
    with pytest.raises(RuntimeError):
        rotate(q.cpu(), None, table, pos)
    with pytest.raises(ValueError):
        RotaryTable(table.cos, table.sin[:, :4])
