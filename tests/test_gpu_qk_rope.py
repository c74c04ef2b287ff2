"""qk_norm_rope and its gradient on the GPU against 64-bit forms and differences."""
import pytest
import torch

import my_own_cnn_b200 as b2q
from lowbit_ref import UNIT, norm_rope, within

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]
EPS = 1e-5


def make(t, hq, hk, d, rot, dtype, fused=False, weights=True, seed=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*s):
        return torch.randn(*s, generator=g, device="cuda")

    if fused:
        x = normal(t, hq + 2 * hk, d).to(dtype)
        q, k = x[:, :hq], x[:, hq:hq + hk]
    else:
        q, k = normal(t, hq, d).to(dtype), normal(t, hk, d).to(dtype)
    qw, kw = ((1 + 0.3 * normal(d)).to(dtype) if weights else None for _ in range(2))
    table = b2q.rope_table(500, rot) if rot else None
    pos = torch.randint(0, 500, (t,), generator=g, device="cuda", dtype=torch.int32) if rot else None
    return q, k, qw, kw, table, pos


def check_side(y, x, w, table, pos, interleaved):
    w = None if w is None else w.double()
    want = norm_rope(x.double(), w, table, pos, EPS, interleaved)
    # the norm's own chain (d / 32 + 5 additions, a square root) and a pair's rotation
    n = norm_rope(x.double(), w, None, None, EPS, interleaved).abs()
    size = n.amax(-1, keepdim=True)
    within(y, want, 1.01 * UNIT[x.dtype] * want.abs() + 2.0 ** -20 * size + (2.0 ** -25 if x.dtype == torch.float16 else 0))


SHAPES = [(1, 1, 1, 64, 64), (1, 32, 8, 128, 128), (3, 7, 1, 80, 80), (5, 4, 4, 96, 48), (33, 5, 2, 256, 256),
          (130, 12, 4, 128, 64), (2, 3, 1, 2, 2), (4, 2, 2, 34, 6), (7, 3, 3, 64, 0), (3, 2, 1, 1000, 500),
          (257, 8, 8, 64, 32), (9, 1, 0, 128, 128), (9, 0, 2, 128, 128), (4, 2, 1, 33, 32)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("t,hq,hk,d,rot", SHAPES)
def test_forward(dtype, interleaved, t, hq, hk, d, rot):
    for fused, weights in ((False, True), (True, True), (True, False)):
        q, k, qw, kw, table, pos = make(t, hq, hk, d, rot, dtype, fused, weights)
        yq, yk = b2q.qk_norm_rope(q, k, qw, kw, table, pos, EPS, interleaved)
        check_side(yq, q, qw, table, pos, interleaved)
        check_side(yk, k, kw, table, pos, interleaved)


@pytest.mark.parametrize("d,rot", [(128, 128), (80, 40), (64, 64)])
def test_in_place_and_odd_alignment(d, rot):
    q, k, qw, kw, table, pos = make(6, 4, 2, d, rot, torch.bfloat16)
    want = b2q.qk_norm_rope(q, k, qw, kw, table, pos, EPS)
    store = torch.zeros(6, 7 * d + 3, device="cuda", dtype=torch.bfloat16)
    vq = store[:, 1:1 + 4 * d].unflatten(1, (4, d))
    vk = store[:, 1 + 4 * d:1 + 6 * d].unflatten(1, (2, d))
    vq.copy_(q)
    vk.copy_(k)
    out = b2q.qk_norm_rope(vq, vk, qw, kw, table, pos, EPS, q_out=vq, k_out=vk)
    assert out[0] is vq and torch.equal(vq, want[0]) and torch.equal(vk, want[1])
    assert (store[:, 0] == 0).all() and (store[:, 1 + 6 * d:] == 0).all()


def test_zero_rows_and_channels_apart():
    q, k, qw, kw, table, pos = make(4, 2, 2, 64, 64, torch.float32)
    q.zero_()
    yq, _ = b2q.qk_norm_rope(q, k, qw, kw, table, pos, EPS)
    assert (yq == 0).all()
    apart = torch.randn(4, 64, 2, device="cuda").transpose(1, 2)
    yq, _ = b2q.qk_norm_rope(apart, k, qw, kw, table, pos, EPS)
    check_side(yq, apart, qw, table, pos, False)


def reference_grads(q, k, qw, kw, table, pos, dq, dk, interleaved):
    out = []
    for x, w, dy in ((q, qw, dq), (k, kw, dk)):
        x = x.double().detach().requires_grad_()
        w = None if w is None else w.double().detach().requires_grad_()
        norm_rope(x, w, table, pos, EPS, interleaved).backward(dy.double())
        out.append((x.grad, None if w is None else w.grad))
    return out


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("t,hq,hk,d,rot", SHAPES + [(1500, 6, 2, 128, 128)])
def test_gradient(dtype, interleaved, t, hq, hk, d, rot):
    q, k, qw, kw, table, pos = make(t, hq, hk, d, rot, dtype, fused=t % 2 == 1, weights=t % 5 != 4)
    g = torch.Generator(device="cuda")
    g.manual_seed(5)
    dq, dk = (torch.randn(x.shape, generator=g, device="cuda").to(dtype) for x in (q, k))
    gq, gk, gqw, gkw = b2q.qk_norm_rope_bprop(dq, dk, q, k, qw, kw, table, pos, EPS, interleaved)
    want = reference_grads(q, k, qw, kw, table, pos, dq, dk, interleaved)
    u = UNIT[dtype]
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0
    for x, w, dy, gx, gw, (wx, ww) in ((q, qw, dq, gq, gqw, want[0]), (k, kw, dk, gk, gkw, want[1])):
        x = x.double()
        r = (x.square().mean(-1, keepdim=True) + EPS).rsqrt()
        dn = dy.double().abs().amax(-1, keepdim=True) * 1.5  # a rotation's part of the gradient is below sqrt(2) of it
        g = dn * (1 if w is None else w.double().abs().amax())
        size = r * (g + x.abs() * r * r * (g * x.abs()).mean(-1, keepdim=True))
        within(gx, wx, 1.01 * u * wx.abs() + 2.0 ** -19 * size + tiny)
        if w is None:
            assert gw is None
        else:
            assert gw.dtype == dtype
            rows = x.shape[0] * x.shape[1]
            bound = 2.0 ** -23 * (rows / 16 + 64) * (dn * x.abs() * r).sum((0, 1))
            within(gw, ww, 1.01 * u * ww.abs() + bound + tiny)


def test_gradient_against_differences():
    """<dy, (f(x + h v) - f(x - h v)) / 2 h> from the forward kernel against <dx, v> from the gradient's; the same
    for a weight.  In fp32 with h = 2^-6 the difference's own error is near 2^-24 / h per unit, and h^2 / 6 of the
    third derivative: 1e-3 of the sum's size covers both."""
    q, k, qw, kw, table, pos = make(6, 3, 2, 64, 32, torch.float32, seed=3)
    g = torch.Generator(device="cuda")
    g.manual_seed(7)
    dq, dk, vq, vk = (torch.randn(x.shape, generator=g, device="cuda") for x in (q, k, q, k))
    vw = torch.randn(64, generator=g, device="cuda")
    gq, gk, gqw, _ = b2q.qk_norm_rope_bprop(dq, dk, q, k, qw, kw, table, pos, EPS)
    h = 2.0 ** -6

    def loss(q, k, qw):
        yq, yk = b2q.qk_norm_rope(q, k, qw, kw, table, pos, EPS)
        return (yq.double() * dq).sum() + (yk.double() * dk).sum()

    for a, b, grad, v in ((loss(q + h * vq, k, qw), loss(q - h * vq, k, qw), gq, vq),
                          (loss(q, k + h * vk, qw), loss(q, k - h * vk, qw), gk, vk),
                          (loss(q, k, qw + h * vw), loss(q, k, qw - h * vw), gqw, vw)):
        terms = grad.double() * v
        assert abs((a - b) / (2 * h) - terms.sum()) < 1e-3 * (1 + terms.square().sum().sqrt() * 4)


def test_gradient_is_the_same_each_time_and_on_a_stream():
    q, k, qw, kw, table, pos = make(2000, 4, 4, 64, 64, torch.bfloat16)
    dq, dk = torch.randn_like(q), torch.randn_like(k)
    want = b2q.qk_norm_rope_bprop(dq, dk, q, k, qw, kw, table, pos)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got = b2q.qk_norm_rope_bprop(dq, dk, q, k, qw, kw, table, pos, stream=s)
    fwd = b2q.qk_norm_rope(q, k, qw, kw, table, pos, stream=s)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    assert torch.equal(fwd[0], b2q.qk_norm_rope(q, k, qw, kw, table, pos)[0])


def test_no_tokens():
    q, k, qw, kw, table, pos = make(0, 4, 2, 64, 64, torch.float32)
    yq, yk = b2q.qk_norm_rope(q, k, qw, kw, table, pos)
    assert yq.shape == (0, 4, 64) and yk.shape == (0, 2, 64)
    gq, gk, gqw, gkw = b2q.qk_norm_rope_bprop(q, k, q, k, qw, kw, table, pos)
    assert gq.shape == (0, 4, 64) and (gqw == 0).all() and (gkw == 0).all()


@pytest.mark.parametrize("d", [64, 80])
def test_positions_outside_the_table_are_reported(d):
    q, k, qw, kw, table, pos = make(4, 2, 1, d, d, torch.float32)
    b2q.device_error()
    yq = torch.full_like(q, 7.0)
    for bad in (500, -1):
        p = pos.clone()
        p[2] = bad
        b2q.qk_norm_rope(q, k, qw, kw, table, p, EPS, q_out=yq)
        with pytest.raises(b2q.B200QError, match="position"):
            b2q.device_error()
        b2q.qk_norm_rope_bprop(q, k, q, k, qw, kw, table, p)
        with pytest.raises(b2q.B200QError, match="position"):
            b2q.device_error()
    check_side(yq[:2], q[:2], qw, table, pos[:2], False)
    b2q.device_error()


def test_refusals():
    q, k, qw, kw, table, pos = make(4, 2, 1, 64, 64, torch.float32)
    with pytest.raises(TypeError, match="q must be"):
        b2q.qk_norm_rope(q.double(), k, qw, kw, table, pos)
    with pytest.raises(TypeError, match="k must be"):
        b2q.qk_norm_rope(q, k.half(), qw, kw, table, pos)
    with pytest.raises(RuntimeError, match="same tokens"):
        b2q.qk_norm_rope(q, k[:3], qw, kw, table, pos)
    with pytest.raises(RuntimeError, match="q_weight"):
        b2q.qk_norm_rope(q, k, qw[:63], kw, table, pos)
    with pytest.raises(RuntimeError, match="even and at most"):
        b2q.qk_norm_rope(q, k, qw, kw, b2q.rope_table(500, 66), pos)
    with pytest.raises(RuntimeError, match="needs positions"):
        b2q.qk_norm_rope(q, k, qw, kw, table, None)
    with pytest.raises(TypeError, match="positions"):
        b2q.qk_norm_rope(q, k, qw, kw, table, pos.long())
    with pytest.raises(RuntimeError, match="q_out"):
        b2q.qk_norm_rope(q, k, qw, kw, table, pos, q_out=q[:2])
    with pytest.raises(RuntimeError, match="dq and dk"):
        b2q.qk_norm_rope_bprop(q[:2], k, q, k, qw, kw, table, pos)
