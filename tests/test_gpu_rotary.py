"""Head norms with rotation, forward and backward, against float64 (needs a B200).

Tolerances count roundings.  One store to T is off by half a step (u = 2^-11
relative for half, 2^-24 for float).  Before it, a value passes a handful of
fp32 operations (row sum over D <= 128 in chains of 8 and a 4-step tree,
rsqrt, three products, two rotations): each at most 2^-24 of the row's largest
magnitude, fewer than 16 of them, so 2^-20 of that magnitude covers them.
"""
import importlib

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

fa = importlib.import_module("tf-custom-flash-attention_b200")
HALF_STEP = {torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def turn64(x, table, pos, interleaved, sign=1.0):
    """x [.., H, D] float64 rotated by the table's rows at pos [..]."""
    if table is None:
        return x
    h = table.shape[1] // 2
    row = table.double()[pos.long()].unsqueeze(-2)
    c, s = row[..., :h], sign * row[..., h:]
    out = x.clone()
    i = torch.arange(h, device=x.device)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + h)
    out[..., a] = x[..., a] * c - x[..., b] * s
    out[..., b] = x[..., b] * c + x[..., a] * s
    return out


def norm64(x, w, eps):
    x = x.double()
    return x if w is None else x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()


def close(got, ref, dtype, scale):
    """|got - ref| <= half a step of ref + 2^-20 of the row's scale (+ half's smallest step)."""
    tol = HALF_STEP[dtype] * ref.abs() + 2.0 ** -20 * scale + (2.0 ** -25 if dtype == torch.float16 else 0.0)
    bad = (got.double() - ref).abs() > tol
    assert not bad.any(), f"{int(bad.sum())} off, worst {float(((got.double() - ref).abs() / tol).max()):.2f} of the tolerance"


CASES = [
    # dtype, batch shape, Hq, Hk, D, rot, halves or neighbours, q weight, k weight, weight dtype, positions
    (torch.float16, (2, 33), 4, 2, 64, 64, False, True, True, torch.float16, False),
    (torch.float16, (1, 1), 1, 1, 128, 128, False, True, True, torch.float32, False),
    (torch.float16, (1, 700), 8, 8, 128, 64, True, True, True, torch.float32, True),
    (torch.float16, (3, 17), 5, 3, 40, 8, False, True, False, torch.float16, True),
    (torch.float16, (64,), 3, 1, 8, 8, True, False, True, torch.float16, True),
    (torch.float16, (2, 9), 2, 7, 104, 96, False, False, False, torch.float16, False),
    (torch.float32, (2, 33), 4, 2, 64, 32, True, True, True, torch.float32, False),
    (torch.float32, (1, 5, 3), 3, 9, 120, 120, False, True, True, torch.float32, True),
    (torch.float32, (2, 130), 6, 1, 128, 128, False, True, True, torch.float32, False),
    (torch.float32, (1, 2), 1, 1, 16, 0, False, True, True, torch.float32, False),
]


def make(case, seed=0):
    dtype, shape, hq, hk, d, rot, inter, qw, kw, wdt, packed = case
    g = torch.Generator(device="cuda").manual_seed(seed + d)
    q = torch.randn(*shape, hq, d, generator=g, device="cuda").to(dtype)
    k = (3 * torch.randn(*shape, hk, d, generator=g, device="cuda")).to(dtype)
    qw = (1 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(wdt) if qw else None
    kw = (1 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(wdt) if kw else None
    table = fa.rotary_table(1000, rot, device="cuda") if rot else None
    pos = torch.randint(0, 1000, shape, generator=g, device="cuda") if packed else None
    where = pos if pos is not None else torch.arange(shape[-1], device="cuda").expand(shape)
    return q, k, qw, kw, table, pos, where, inter


@pytest.mark.parametrize("case", CASES)
def test_forward(case):
    q, k, qw, kw, table, pos, where, inter = make(case)
    outs = fa.qk_norm_rope(q, k, qw, kw, table, pos, eps=1e-5, interleaved=inter)
    for x, w, y in zip((q, k), (qw, kw), outs):
        ref = turn64(norm64(x, w, 1e-5), table, where, inter)
        assert y.shape == x.shape and y.dtype == x.dtype and y.is_contiguous()
        close(y, ref, x.dtype, ref.abs().amax(-1, keepdim=True))
    assert fa.device_status() == 0


@pytest.mark.parametrize("case", CASES)
def test_backward(case):
    q, k, qw, kw, table, pos, where, inter = make(case, 50)
    g = torch.Generator(device="cuda").manual_seed(7)
    dq_out, dk_out = (torch.randn(x.shape, generator=g, device="cuda").to(x.dtype) for x in (q, k))
    dq, dk, dqw, dkw = fa.qk_norm_rope_grad(q, k, dq_out, dk_out, qw, kw, table, pos, eps=1e-5, interleaved=inter)
    for x, w, dy, dx, dw in ((q, qw, dq_out, dq, dqw), (k, kw, dk_out, dk, dkw)):
        gr = turn64(dy.double(), table, where, inter, -1.0)
        if w is None:
            assert dw is None
            close(dx, gr, x.dtype, gr.abs().amax(-1, keepdim=True))
            continue
        x64 = x.double()
        r = torch.rsqrt((x64 * x64).mean(-1, keepdim=True) + 1e-5)
        n, gw = x64 * r, gr * w.double()
        ref = r * (gw - n * (gw * n).mean(-1, keepdim=True))
        # the projection subtracts terms of the size of r * gw and r * n * mean|gw n|
        size = r * (gw.abs().amax(-1, keepdim=True) + n.abs().amax(-1, keepdim=True) * (gw * n).abs().mean(-1, keepdim=True))
        close(dx, ref, x.dtype, size)
        terms = (gr * n).flatten(0, -2)
        # each term carries under 8 fp32 roundings, and is added in a chain of (rows of a lane) < 64 and 48 more
        tol = 128 * 2.0 ** -24 * terms.abs().sum(0) + (HALF_STEP[w.dtype] * terms.sum(0).abs())
        assert ((dw.double() - terms.sum(0)).abs() <= tol).all()
        assert dw.dtype == w.dtype
    assert fa.device_status() == 0


def test_gradient_against_differences():
    """The gradient of a float64 model of the op by central differences, at a few places, against the kernel's."""
    case = (torch.float32, (2, 3), 2, 1, 16, 8, False, True, True, torch.float32, False)
    q, k, qw, kw, table, pos, where, inter = make(case)
    q, k, qw, kw = (x.requires_grad_() for x in (q, k, qw, kw))
    g = torch.Generator(device="cuda").manual_seed(1)
    cq, ck = (torch.randn(x.shape, generator=g, device="cuda") for x in (q, k))
    yq, yk = fa.autograd.qk_norm_rope(q, k, qw, kw, table, eps=1e-5)
    grads = torch.autograd.grad((yq * cq).sum() + (yk * ck).sum(), (q, k, qw, kw))

    def loss(vals):
        a, b, u, v = vals
        return float((turn64(norm64(a, u, 1e-5), table, where, False) * cq.double()).sum()
                     + (turn64(norm64(b, v, 1e-5), table, where, False) * ck.double()).sum())

    base = [x.detach().double() for x in (q, k, qw, kw)]
    step = 1e-4
    for i in range(4):
        for j in range(0, base[i].numel(), 5):
            up, dn = [x.clone() for x in base], [x.clone() for x in base]
            up[i].view(-1)[j] += step
            dn[i].view(-1)[j] -= step
            fd = (loss(up) - loss(dn)) / (2 * step)
            # third derivatives of x * rsqrt(mean x^2) are O(|c| / |x|^2): step^2 = 1e-8 of O(100); fp32 2^-18 of O(10)
            assert abs(float(grads[i].view(-1)[j]) - fd) <= 2e-4


def test_strided_inputs_and_shared_weight():
    """Slices of a fused projection are read in place; one weight for both sides gets the sum of its gradients."""
    B, S, H, D = 2, 37, 4, 64
    g = torch.Generator(device="cuda").manual_seed(3)
    fused = torch.randn(B, S, 3 * H * D, generator=g, device="cuda").half()
    q, k = fused[..., : H * D].view(B, S, H, D), fused[..., H * D: 2 * H * D].view(B, S, H, D)
    w = (1 + 0.1 * torch.randn(D, generator=g, device="cuda"))
    table = fa.rotary_table(S, D, device="cuda")
    got = fa.qk_norm_rope(q, k, w, w, table)
    ref = fa.qk_norm_rope(q.contiguous(), k.contiguous(), w, w, table)
    assert all(torch.equal(a, b) for a, b in zip(got, ref))
    heads_apart = torch.randn(B, H, S, D, generator=g, device="cuda").half().transpose(1, 2)  # heads not dense: copied
    one_row = torch.randn(1, 1, H, D, generator=g, device="cuda").half().expand(B, S, H, D)  # stride 0: copied
    got = fa.qk_norm_rope(heads_apart, one_row, w, w, table)
    ref = fa.qk_norm_rope(heads_apart.contiguous(), one_row.contiguous(), w, w, table)
    assert all(torch.equal(a, b) for a, b in zip(got, ref))
    odd = torch.randn(B * S * H * D + 1, generator=g, device="cuda").half()[1:].view(B, S, H, D)  # 2 bytes off
    assert torch.equal(fa.qk_norm_rope(odd, odd, w, w, table)[0], fa.qk_norm_rope(odd.clone(), odd.clone(), w, w, table)[0])
    w = w.requires_grad_()
    q1 = q.detach().clone().requires_grad_()
    yq, yk = fa.autograd.qk_norm_rope(q1, q1, w, w, table)
    gq, gw = torch.autograd.grad((yq.float().sum() + 2 * yk.float().sum()), (q1, w))
    one = torch.ones_like(yq)
    a = fa.qk_norm_rope_grad(q1.detach(), q1.detach(), one, 2 * one, w.detach(), w.detach(), table)
    assert torch.equal(gw, a[2] + a[3]) and torch.equal(gq, a[0] + a[1])


def test_sides_of_other_lengths_and_empty_ones():
    D = 32
    table = fa.rotary_table(64, D, device="cuda")
    q, k = torch.randn(2, 5, 3, D, device="cuda"), torch.randn(2, 40, 1, D, device="cuda")
    w = torch.ones(D, device="cuda")
    yq, yk = fa.qk_norm_rope(q, k, w, w, table)
    for x, y in ((q, yq), (k, yk)):
        ref = turn64(norm64(x, w, 1e-6), table, torch.arange(x.shape[1], device="cuda").expand(2, -1), False)
        close(y, ref, x.dtype, ref.abs().amax(-1, keepdim=True))
    e = torch.randn(2, 0, 3, D, device="cuda")
    yq, yk = fa.qk_norm_rope(e, k, w, w, table)
    assert yq.shape == e.shape and yk.shape == k.shape
    dq, dk, dqw, dkw = fa.qk_norm_rope_grad(e, e, e, e, w, w, table)
    assert dq.shape == e.shape and not dqw.any() and not dkw.any()


def test_positions_outside_the_table_are_clamped_and_reported():
    D = 16
    table = fa.rotary_table(8, D, device="cuda")
    q = torch.randn(1, 4, 1, D, device="cuda")
    pos = torch.tensor([[-3, 0, 7, 900]], device="cuda")
    fa.device_status()
    y, _ = fa.qk_norm_rope(q, q, table=table, q_positions=pos)
    assert fa.device_status() == 2
    ref, _ = fa.qk_norm_rope(q, q, table=table, q_positions=pos.clamp(0, 7))
    assert torch.equal(y, ref) and fa.device_status() == 0


@pytest.mark.parametrize("far", [2 ** 32 + 3, -(2 ** 32) + 3, 2 ** 31, 2 ** 62])
def test_wide_positions_are_not_cut_to_a_row_of_the_table(far):
    table = fa.rotary_table(8, 64)
    q = torch.randn(1, 2, 2, 64, device="cuda")
    fa.device_status()
    y, _ = fa.qk_norm_rope(q, q, table=table, q_positions=torch.tensor([[1, far]], device="cuda"))
    assert fa.device_status() == 2
    ref, _ = fa.qk_norm_rope(q, q, table=table, q_positions=torch.tensor([[1, 0 if far < 0 else 7]], device="cuda"))
    assert torch.equal(y, ref) and fa.device_status() == 0


def test_far_positions():
    """Angles of 10^5 radians: the table is taken in float64."""
    table = fa.rotary_table(131072, 64, device="cuda")
    pos = torch.tensor([131071, 99999, 3], dtype=torch.float64)
    inv = 10000.0 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64)
    ang = pos[:, None] * inv
    ref = torch.cat([ang.cos(), ang.sin()], 1)
    assert (table[pos.long()].cpu().double() - ref).abs().max() <= 2.0 ** -24


def test_same_bits_every_run_on_two_streams_and_in_a_graph():
    case = (torch.float16, (4, 900), 8, 4, 128, 128, False, True, True, torch.float32, False)
    q, k, qw, kw, table, pos, where, inter = make(case)
    dq_out, dk_out = torch.randn_like(q), torch.randn_like(k)
    torch.cuda.synchronize()

    def step():
        return [*fa.qk_norm_rope(q, k, qw, kw, table), *fa.qk_norm_rope_grad(q, k, dq_out, dk_out, qw, kw, table)]

    ref = step()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs.append(step())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    new = torch.randn_like(q)
    ref_new = None
    old = q.clone()
    q.copy_(new)
    graph.replay()
    torch.cuda.synchronize()
    ref_new = step()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(captured, ref_new))
    q.copy_(old)
    graph.replay()
    torch.cuda.synchronize()
    for o in (*outs, captured):
        assert all(torch.equal(a, b) for a, b in zip(o, ref))


@pytest.mark.parametrize("dtype,shape,hq,hk,d,rot,inter", [
    (torch.float16, (3, 6500), 3, 1, 128, 128, False),   # a group walks several tokens: the loads run ahead
    (torch.float16, (1, 40000), 1, 2, 40, 24, True),
    (torch.float32, (2, 9700), 3, 2, 64, 32, False),
])
def test_long_inputs(dtype, shape, hq, hk, d, rot, inter):
    """Forward and backward over more tokens than the backward's groups."""
    case = (dtype, shape, hq, hk, d, rot, inter, True, True, torch.float32, True)
    q, k, qw, kw, table, pos, where, _ = make(case, 4)
    for x, w, y in zip((q, k), (qw, kw), fa.qk_norm_rope(q, k, qw, kw, table, pos, eps=1e-5, interleaved=inter)):
        ref = turn64(norm64(x, w, 1e-5), table, where, inter)
        close(y, ref, x.dtype, ref.abs().amax(-1, keepdim=True))
    g = torch.Generator(device="cuda").manual_seed(8)
    dys = [torch.randn(x.shape, generator=g, device="cuda").to(dtype) for x in (q, k)]
    grads = fa.qk_norm_rope_grad(q, k, *dys, qw, kw, table, pos, eps=1e-5, interleaved=inter)
    for x, w, dy, dx, dw in ((q, qw, dys[0], grads[0], grads[2]), (k, kw, dys[1], grads[1], grads[3])):
        gr = turn64(dy.double(), table, where, inter, -1.0)
        x64 = x.double()
        r = torch.rsqrt((x64 * x64).mean(-1, keepdim=True) + 1e-5)
        n, gw = x64 * r, gr * w.double()
        size = r * (gw.abs().amax(-1, keepdim=True) + n.abs().amax(-1, keepdim=True) * (gw * n).abs().mean(-1, keepdim=True))
        close(dx, r * (gw - n * (gw * n).mean(-1, keepdim=True)), dtype, size)
        terms = (gr * n).flatten(0, -2)
        # a lane adds under 64 rows here, the tree behind it 48 more: see test_backward
        assert ((dw.double() - terms.sum(0)).abs() <= 128 * 2.0 ** -24 * terms.abs().sum(0) + 2.0 ** -24 * terms.sum(0).abs()).all()
    assert fa.device_status() == 0
