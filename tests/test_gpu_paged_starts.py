"""Starts (q_start) that descend or leave the call's tokens: reported, and out of memory (needs a B200)."""
import importlib

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

fa = importlib.import_module("tf-custom-flash-attention_b200")
base = importlib.import_module("test_gpu_paged")
H16, F32 = torch.float16, torch.float32


def step(dtype, T, starts, held, hq, hkv, d=64, page=16):
    """T tokens over sequences that all read the same pages."""
    g = torch.Generator(device="cuda").manual_seed(T)
    n, m = len(starts) - 1, -(-held // page)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dtype)
    return dict(q=r(T, hq, d), k_pages=r(m + 2, page, hkv, d), v_pages=r(m + 2, page, hkv, d),
                page_table=torch.arange(m, dtype=torch.int32, device="cuda").expand(n, m).contiguous(),
                kv_len=torch.full((n,), held, dtype=torch.int32, device="cuda"),
                q_start=torch.tensor(starts, dtype=torch.int32, device="cuda"))


DESCENDING = [
    (H16, 1024, [0, 1024] * 20 + [0], 1024, 32, 8),       # chunks: more items than the launch has CTAs
    (H16, 4096, [0, 4096] * 6 + [0], 4096, 8, 8),
    (H16, 300, [0, 300, 0, 300], 300, 2, 1),              # fewer items than SMs
    (H16, 300, [0, 5, 3, 300], 300, 2, 1),
    (H16, 200, [0] + [200, 0] * 50, 200, 4, 2),           # over 32 sequences
    (H16, 9, [0, 9, 2, 5, 9, 9, 9, 9, 9, 9], 40, 4, 2),   # few rows
    (H16, 130, [130, 0] * 130 + [7], 77, 4, 4),           # over 128 sequences
    (F32, 40, [0, 40, 0, 40], 60, 4, 2),
    (F32, 3, [3, 2, 1, 0], 33, 1, 1),
    (F32, 200, [-5, 200, -2 ** 31, 2 ** 31 - 1, 0], 200, 2, 2),
]


@pytest.mark.parametrize("case", DESCENDING)
@pytest.mark.parametrize("causal", [True, False])
def test_shared_tokens_leave_the_call_out(case, causal):
    dtype, T, starts, held, hq, hkv = case
    s = step(*case)
    fa.device_status()
    out, stats = torch.full_like(s["q"], 7.0), torch.full((T, hq), 7.0, device="cuda")
    fa.paged_sdpa(**s, out=(out, stats), scale=0.125, causal_mask=causal)
    assert fa.device_status() == 2
    assert (out == 7).all() and (stats == 7).all()
    lens = [(T, max(T, held))]  # the same memory, starts in order
    good = step(dtype, T, [0, T], max(T, held), hq, hkv)
    base.check_attend(good, lens, 0.125, causal, fa.paged_sdpa(**good, scale=0.125, causal_mask=causal))
    assert fa.device_status() == 0


@pytest.mark.parametrize("dtype,T,hq", [(H16, 5, 2), (H16, 300, 4), (H16, 200, 130), (F32, 5, 1), (F32, 90, 4)])
@pytest.mark.parametrize("empty", [0, 40, 200])
def test_descending_starts_that_share_nothing(dtype, T, hq, empty):
    """Unused places of a batch left at zero: empty to the attention, whose rows are those of the used ones; reported."""
    lens = [(2, 40), (T - 2, T + 30)] + [(0, 50)] * (empty + 1)
    s = base.make(dtype, lens, hq, 2 if hq == 4 else 1, 64, 64, 16, seed=3)
    want = fa.paged_sdpa(**s, scale=0.125)
    assert fa.device_status() == 0
    s["q_start"][3:] = 0
    got = fa.paged_sdpa(**s, scale=0.125)
    assert fa.device_status() == 2
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("case", DESCENDING)
def test_descending_starts_write_inside_their_pages(case):
    dtype, T, starts, held, hq, hkv = case
    s = step(*case)
    fa.device_status()
    before = s["k_pages"].clone(), s["v_pages"].clone()
    k = torch.randn(T, hkv, 64, device="cuda").to(dtype)
    q = fa.paged_append(k, k, s["k_pages"], s["v_pages"], s["page_table"], s["kv_len"], s["q_start"], q=s["q"])
    assert fa.device_status() == 2 and q.shape == s["q"].shape
    for a, b in zip((s["k_pages"], s["v_pages"]), before):
        assert torch.equal(a[-2:], b[-2:])  # (in no sequence's table)


@pytest.mark.parametrize("dtype,T", [(H16, 6), (H16, 200), (F32, 6), (F32, 50)])
@pytest.mark.parametrize("first,last", [(0, 5), (-3, 0), (-2 ** 31, 2 ** 30)])
def test_starts_outside_the_call_are_clamped(dtype, T, first, last):
    """The write and the attention place every token alike: as if the starts ended with the call's tokens."""
    lens = [(3, 40), (0, 17), (T - 3, T + 30)]
    got = []
    for lo, over in ((0, 0), (first, last)):
        s = base.make(dtype, lens, 4, 2, 64, 64, 16, seed=3)
        assert s["q_start"].tolist() == [0, 3, 3, T]
        s["q_start"][0], s["q_start"][3] = lo, T + over
        g = torch.Generator(device="cuda").manual_seed(1)
        k, v = (torch.randn(T, 2, 64, generator=g, device="cuda").to(dtype) for _ in range(2))
        table = fa.rotary_table(T + 64, 64)
        fa.device_status()
        s["q"] = fa.paged_append(k, v, s["k_pages"], s["v_pages"], s["page_table"], s["kv_len"], s["q_start"], q=s["q"], table=table)
        assert fa.device_status() == (0 if (lo, over) == (0, 0) else 2)
        got.append((s["q"], s["k_pages"].nan_to_num(9), s["v_pages"].nan_to_num(9), *fa.paged_sdpa(**s, scale=0.125)))
        assert fa.device_status() == (0 if (lo, over) == (0, 0) else 2)
    assert all(torch.equal(a, b) for a, b in zip(*got))
