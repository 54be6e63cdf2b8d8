"""paged_sdpa in float: values of any magnitude, and the statistics of a whole serving run (needs a B200).

The bounds are those of test_gpu_paged (roundings counted there); they are relative to the sums of magnitudes,
so they hold at any scale as long as nothing leaves float's range."""
import importlib

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

fa = importlib.import_module("tf-custom-flash-attention_b200")
base = importlib.import_module("test_gpu_paged")

BIG = 2.0 ** 116  # 8.3e34; |randn| < 6, and a row's 300 unnormalised weights are at most 1 each: sums stay below 1.6e38


@pytest.mark.parametrize("new", [1, 9, 40])  # 8-row tiles, pairs of 16, four of 16
@pytest.mark.parametrize("d,dv", [(64, 64), (128, 96)])
@pytest.mark.parametrize("large", ["q", "k", "v", "all"])
def test_large_float_values(new, d, dv, large):
    """Queries, keys or values past 2^115; where scores would leave the range the other factor or the scale is small."""
    lens = [(new, 300), (new, 44)]
    s = base.make(torch.float32, lens, 4, 2, d, dv, 16, seed=7)
    scale = d ** -0.5
    if large == "q":
        s["q"] *= BIG
        s["k_pages"] *= 2.0 ** -90
        scale *= 2.0 ** -26
    elif large == "k":
        s["k_pages"] *= BIG
        scale *= 2.0 ** -116
    else:
        s["v_pages"] *= BIG
        if large == "all":
            s["q"] *= 2.0 ** -90
            s["k_pages"] *= BIG
            scale *= 2.0 ** -26
    base.check_attend(s, lens, scale, True, fa.paged_sdpa(**s, scale=scale))
    assert fa.device_status() == 0


def test_float_statistics_of_a_prompt_then_tokens():
    """The statistics of a prompt in two chunks and then tokens against one causal call of sdpa over the whole: each
    side is off by at most ds + 2^-21 (1 + |stats|) (see test_gpu_paged), with ds = 2^-20 scale sum|q||k| +
    2^-22 (1 + 2 max|x|); the two together by twice that."""
    H, D, S, page, B = 4, 64, 300, 16, 2
    g = torch.Generator(device="cuda").manual_seed(11)
    q, k, v = (torch.randn(B, S, H, D, generator=g, device="cuda") for _ in range(3))
    qw, kw = (1 + 0.1 * torch.randn(D, generator=g, device="cuda") for _ in range(2))
    table = fa.rotary_table(S, D, device="cuda")
    rq, rk = fa.qk_norm_rope(q, k, qw, kw, table)
    _, dense = fa.sdpa_bshd(rq, rk, v, 0, 0, scale=D ** -0.5, causal_mask=True)
    pages = -(-S // page)
    k_pages = torch.full((B * pages, page, H, D), float("nan"), device="cuda")
    v_pages = k_pages.clone()
    pt = torch.randperm(B * pages, generator=torch.Generator().manual_seed(0)).int().view(B, pages).cuda()
    stats, at = torch.zeros(B, H, S, device="cuda"), 0
    for step in [170, 125, 1, 1, 3]:
        x = [t[:, at:at + step].reshape(B * step, H, D) for t in (q, k, v)]
        at += step
        kv_len = torch.full((B,), at, dtype=torch.int32, device="cuda")
        q_start = torch.arange(B + 1, dtype=torch.int32, device="cuda") * step
        qq = fa.paged_append(x[1], x[2], k_pages, v_pages, pt, kv_len, q_start, q=x[0], q_weight=qw, k_weight=kw, table=table)
        _, st = fa.paged_sdpa(qq, k_pages, v_pages, pt, kv_len, q_start, scale=D ** -0.5)
        stats[:, :, at - step:at] = st.view(B, step, H).transpose(1, 2)
    x = torch.einsum("bihd,bjhd->bhij", rq.double(), rk.double()) * D ** -0.5
    ds = torch.einsum("bihd,bjhd->bhij", rq.double().abs(), rk.double().abs()) * D ** -0.5
    dead = torch.ones(S, S, dtype=torch.bool, device="cuda").triu(1)
    big = x.masked_fill(dead, 0).abs().amax(-1)
    x = x.masked_fill(dead, -float("inf"))
    m = x.amax(-1)
    ref = m + torch.log(torch.exp(x - m[..., None]).sum(-1) + 1e-6)
    tol = 2.0 ** -20 * ds.amax(-1) + 2.0 ** -22 * (1 + 2 * big) + 2.0 ** -21 * (1 + ref.abs())
    for got, bound in ((stats.double() - ref, tol), (dense.view(B, H, S).double() - stats.double(), 2 * tol)):
        assert (got.abs() <= bound).all(), f"worst {float((got.abs() / bound).max()):.2f} of the tolerance"
    assert fa.device_status() == 0
