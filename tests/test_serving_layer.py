"""The layer's norms and rotation, its paged form, and the cache's accounting."""
import importlib

import pytest

torch = pytest.importorskip("torch")

fa = importlib.import_module("tf-custom-flash-attention_b200")


def test_cache_accounting():
    c = fa.PagedCache(6, 16, 2, 8, device="cpu")
    b = c.batch([("a", 17), ("b", 0), ("c", 16)])
    assert b.tokens == 33 and b.q_start.tolist() == [0, 17, 17, 33] and b.kv_len.tolist() == [17, 0, 16]
    assert b.page_table.shape == (3, 2) and b.page_table[1].tolist() == [-1, -1]
    used = [x for x in b.page_table.flatten().tolist() if x >= 0]
    assert len(used) == len(set(used)) == 3
    b2 = c.batch([("c", 1), ("a", 15)])
    assert b2.kv_len.tolist() == [17, 32] and c.length("a") == 32
    assert b2.page_table[1].tolist() == b.page_table[0].tolist()  # 32 tokens still fit its two pages
    with pytest.raises(fa.InvalidArgumentError, match="2 free pages, the batch needs 3"):
        c.batch([("d", 48)])
    with pytest.raises(fa.InvalidArgumentError, match="once"):
        c.batch([("a", 1), ("a", 1)])
    with pytest.raises(fa.InvalidArgumentError, match="negative"):
        c.batch([("a", -1)])
    assert c.length("a") == 32 and c.length("d") == 0  # refused batches reserve nothing
    c.free("a")
    c.free("nobody")
    assert c.length("a") == 0 and c.batch([("d", 64)]).page_table.shape == (1, 4)
    assert c.batch([]).q_start.tolist() == [0]


def test_layer_arguments():
    with pytest.raises(ValueError, match="max_positions"):
        fa.MHA(num_heads=2, rotary_dim=16)
    assert not fa.MHA(num_heads=2).state_dict()  # the extensions are off by default
    assert set(fa.MHA(num_heads=2, qk_norm_dim=16).state_dict()) == {"q_norm", "k_norm"}


def dense64(m, q, k, v, H, causal):
    """The layer in float64: norm, rotation (pairs i, i + rot/2), softmax(q k^T / sqrt(D)) v over [B, S, H*D]."""
    B, S, F = q.shape
    D = F // H
    x = [t.double().view(B, t.shape[1], H, -1) for t in (q, k, v)]
    for i, w in ((0, m.q_norm), (1, m.k_norm)):
        if w is not None:
            x[i] = x[i] * torch.rsqrt((x[i] ** 2).mean(-1, keepdim=True) + 1e-6) * w.double()
        if m.rotary_dim:
            h = m.rotary_dim // 2
            ang = torch.arange(x[i].shape[1], device=q.device, dtype=torch.float64)[:, None] * m.rotary_base ** (
                -torch.arange(h, device=q.device, dtype=torch.float64) / h)
            c, s = ang.cos()[:, None], ang.sin()[:, None]
            a, b = x[i][..., :h], x[i][..., h:2 * h]
            x[i] = torch.cat([a * c - b * s, b * c + a * s, x[i][..., 2 * h:]], -1)
    sc = torch.einsum("bihd,bjhd->bhij", x[0], x[1]) * D ** -0.5
    if causal:
        sc = sc.masked_fill(torch.ones_like(sc, dtype=torch.bool).triu(1), -float("inf"))
    return torch.einsum("bhij,bjhe->bihe", sc.softmax(-1), x[2]).reshape(B, S, -1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,layout,rot", [(torch.float16, "bsf", 64), (torch.float32, "bsf", 32), (torch.float16, "sbf", 64)])
def test_layer_with_norm_and_rotation_and_its_gradients(dtype, layout, rot):
    """Against the layer in float64 and autograd through it.  Tolerances, relative to the largest value of each
    result: half 4e-3 forward and 1e-2 gradients (the attention's own 2e-3 on inputs rounded once more, 2^-11, then
    through the norm's gradient); float 1e-5 and 3e-5."""
    torch.manual_seed(1)
    B, S, H, D = 2, 130, 3, 64
    ax = -2 if layout == "bsf" else 0
    m = fa.MHA(num_heads=H, seq_axis=ax, causal_mask=True, qk_norm_dim=D, rotary_dim=rot, rotary_base=5000.0,
               max_positions=256).cuda().train()
    with torch.no_grad():
        m.q_norm.add_(0.2 * torch.randn(D, device="cuda")), m.k_norm.add_(0.2 * torch.randn(D, device="cuda"))
    x = [torch.randn(B, S, H * D, device="cuda").to(dtype).requires_grad_() for _ in range(3)]
    give = (lambda t: t) if layout == "bsf" else (lambda t: t.transpose(0, 1))
    out = give(m(*[give(t) for t in x]))
    go = torch.randn_like(out)
    grads = torch.autograd.grad(out, (*x, m.q_norm, m.k_norm), go)
    y = [t.detach().double().requires_grad_() for t in x]
    ref = dense64(m, *y, H, True)
    ref_grads = torch.autograd.grad(ref, (*y, m.q_norm, m.k_norm), go.double())
    tol_o, tol_g = (4e-3, 1e-2) if dtype == torch.float16 else (1e-5, 3e-5)
    assert (out.double() - ref).abs().max() <= tol_o * ref.abs().max()
    for a, b in zip(grads, ref_grads):
        assert (a.double() - b.double()).abs().max() <= tol_g * b.abs().max()
    assert fa.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("kv_heads", [4, 2])
@pytest.mark.parametrize("extras", [True, False])
def test_paged_layer_answers_like_the_whole_sequence(kv_heads, extras):
    """Prompts of three users in chunks, then tokens, through MHA.forward_paged; against the float64 layer."""
    torch.manual_seed(2)
    H, D = 4, 64
    kw = dict(qk_norm_dim=D, rotary_dim=D, max_positions=512) if extras else {}
    m = fa.MHA(num_heads=H, causal_mask=True, **kw).cuda().eval().requires_grad_(False)
    lens = {"x": 150, "y": 33, "z": 300}
    q = {s: torch.randn(n, H * D, device="cuda").half() for s, n in lens.items()}
    k = {s: torch.randn(n, kv_heads * D, device="cuda").half() for s, n in lens.items()}
    v = {s: torch.randn(n, kv_heads * D, device="cuda").half() for s, n in lens.items()}
    cache = fa.PagedCache(40, 16, kv_heads, D)
    outs = {s: [] for s in lens}
    for step in ([("x", 100), ("y", 32)], [("z", 290), ("x", 49), ("y", 0)], [("y", 1), ("x", 1), ("z", 5)], [("z", 5)]):
        at = {s: cache.length(s) for s, _ in step}
        batch = cache.batch(step)
        cat = [torch.cat([t[s][at[s]:at[s] + n] for s, n in step]) for t in (q, k, v)]
        o = m.forward_paged(*cat, cache, batch).split([n for _, n in step])
        for (s, _), part in zip(step, o):
            outs[s].append(part)
    assert fa.device_status() == 0
    rep = H // kv_heads
    for s, n in lens.items():
        wide = [t[s].view(n, kv_heads, 1, D).expand(n, kv_heads, rep, D).reshape(1, n, H * D) for t in (k, v)]
        ref = dense64(m, q[s][None], *wide, H, True)[0]
        got = torch.cat(outs[s])
        assert got.shape == ref.shape and (got.double() - ref).abs().max() <= 4e-3 * ref.abs().max()
    for s in lens:
        cache.free(s)
    assert len(cache._free) == 40


@pytest.mark.gpu
def test_captured_training_step():
    """Forward and gradients captured; replays follow new inputs.  (No eager graph of the same leaves may live then:
    torch joins the capture with the stream of the leaves' old accumulation nodes and invalidates it, whatever the
    operator.)"""
    torch.manual_seed(3)
    q = torch.randn(2, 50, 4, 64, device="cuda").half().requires_grad_()
    w = torch.ones(64, device="cuda").requires_grad_()
    table = fa.rotary_table(64, 64)
    go = torch.randn(2, 50, 4, 64, device="cuda").half()

    def step():
        a, b = fa.autograd.qk_norm_rope(q, q, w, w, table)
        return torch.autograd.grad((a, b), (q, w), (go, go))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    with torch.no_grad():
        q.copy_(torch.randn_like(q))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(captured, step()))


@pytest.mark.gpu
def test_layer_refuses_to_lay_out_its_table_in_a_capture():
    m = fa.MHA(num_heads=1, rotary_dim=64, max_positions=64).cuda().eval()
    x = torch.randn(1, 8, 64, device="cuda").half()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="before capturing"):
        with torch.cuda.graph(graph):
            m(x, x, x)
    torch.cuda.synchronize()
    with pytest.raises(ValueError, match="max_positions"):
        m(*[torch.randn(1, 65, 64, device="cuda").half()] * 3)
    assert m(x, x, x).shape == x.shape
