"""The paged cache: its write and the attention over it, against float64 (needs a B200).

Tolerances count roundings, u = 2^-11 (half) or 2^-24 (float) for half a step.
Attention: with A = sum_j softmax_j |v_j| and n keys,
  half:  P enters the product in half, off by u relative or 2^-25 (below half's
         normal range; the largest p of a row is 1, so l >= 1):
         u |o| (the store) + u A + n 2^-25 max|v|;
  both:  a score is off by ds = scale * sum|q||k| * e, e = 2^-17 for half (exact
         products, 128 sums of at most 2^-24 each) and 2^-20 for float (three
         tf32 products of 2^-22 and short sums), an exponential by 2^-21 and by
         its argument's rounding 2^-23 |x|, |x| <= 64 counted (smaller p add
         nothing), so p is off by ds + 2^-16 at most, and the quotient by twice
         that: 2 (ds + 2^-16) A for half; for float the argument's share is
         counted from the scores at hand, 2 (ds + 2^-22 (1 + max|x|)) A.
stats: ds + 2^-21 (1 + |stats|) and the half bound's 2^-16 replaced likewise.
"""
import importlib

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

fa = importlib.import_module("tf-custom-flash-attention_b200")
HALF_STEP = {torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def make(dtype, lens, hq, hkv, d, dv, page, seed=0, tail=0, amp=1.0):
    """lens: (new, held) of each sequence; unused pool rows are NaN, unused table entries out of range."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    used = [-(-h // page) for _, h in lens]
    pool = sum(used) + 1
    ids = torch.randperm(pool, generator=torch.Generator().manual_seed(seed)).tolist()
    width = max(used + [1]) + 1
    k_pages = torch.full((pool, page, hkv, d), float("nan"), device="cuda", dtype=dtype)
    v_pages = torch.full((pool, page, hkv, dv), float("nan"), device="cuda", dtype=dtype)
    table = torch.full((len(lens), width), 2 ** 30, dtype=torch.int32)
    for n, (_, h) in enumerate(lens):
        for i in range(used[n]):
            p = ids.pop()
            table[n, i] = p
            rows = min(page, h - i * page)
            k_pages[p, :rows] = torch.randn(rows, hkv, d, generator=g, device="cuda").to(dtype)
            v_pages[p, :rows] = torch.randn(rows, hkv, dv, generator=g, device="cuda").to(dtype)
    start = [0]
    for a, _ in lens:
        start.append(start[-1] + a)
    T = start[-1] + tail
    q = (amp * torch.randn(T, hq, d, generator=g, device="cuda")).to(dtype)
    return dict(q=q, k_pages=k_pages, v_pages=v_pages, page_table=table.cuda(),
                kv_len=torch.tensor([h for _, h in lens], dtype=torch.int32, device="cuda"),
                q_start=torch.tensor(start, dtype=torch.int32, device="cuda"))


def gather(s, n, held):
    page = s["k_pages"].shape[1]
    j = torch.arange(held, device="cuda")
    slots = s["page_table"][n].long()[j // page] * page + j % page
    return s["k_pages"].flatten(0, 1)[slots].double(), s["v_pages"].flatten(0, 1)[slots].double()


def check_attend(s, lens, scale, causal, got, skip=()):
    out, stats = got
    dtype, (T, hq, d) = s["q"].dtype, s["q"].shape
    hkv = s["k_pages"].shape[2]
    G, at = hq // hkv, 0
    for n, (new, held) in enumerate(lens):
        if new and n not in skip:
            k, v = gather(s, n, held)
            q = s["q"][at:at + new].double().view(new, hkv, G, d)
            x = torch.einsum("thgd,jhd->thgj", q, k) * scale
            ds = (torch.einsum("thgd,jhd->thgj", q.abs(), k.abs()) * abs(scale)).amax(-1) if held else torch.zeros(new, hkv, G).cuda()
            j, i = torch.arange(held, device="cuda"), torch.arange(new, device="cuda")
            lim = (held - new + i + 1 if causal else torch.full_like(i, held)).clamp(0, held)
            dead = (j[None] >= lim[:, None])[:, None, None]
            big = x.masked_fill(dead, 0).abs().amax(-1) if held else ds
            x = x.masked_fill(dead, -float("inf"))
            m = x.amax(-1).clamp_min(-1e9) if held else torch.full((new, hkv, G), -1e9, dtype=torch.float64, device="cuda")
            p = torch.exp(x - m[..., None])
            l = p.sum(-1)
            ref_s = (m + torch.log(l + 1e-6)).view(new, hq)
            w = p / l.clamp_min(1e-300)[..., None]
            ref = torch.einsum("thgj,jhe->thge", w, v).reshape(new, hq, -1)
            A = torch.einsum("thgj,jhe->thge", w, v.abs()).reshape(new, hq, -1)
            u = HALF_STEP[dtype]
            if dtype == torch.float16:
                dp = ds * 2.0 ** -17 + 2.0 ** -16
                vmax = float(v.abs().max()) if held else 0.0
                tol = u * ref.abs() + u * A + held * 2.0 ** -25 * vmax + 2 * dp.reshape(new, hq, 1) * A + 2.0 ** -25
            else:
                dp = ds * 2.0 ** -20 + 2.0 ** -22 * (1 + 2 * big)
                tol = u * ref.abs() + 2 * dp.reshape(new, hq, 1) * A
            a = out[at:at + new].double()
            err = (a - ref).abs()
            assert torch.isfinite(a).all(), f"sequence {n}"
            assert (err <= tol).all(), f"sequence {n}: worst {float((err / tol.clamp_min(1e-300)).max()):.2f} of the tolerance"
            es = (stats[at:at + new].double() - ref_s).abs()
            ts = dp.reshape(new, hq) + 2.0 ** -21 * (1 + ref_s.abs())
            assert (es <= ts).all(), f"sequence {n}: stats {float((es / ts).max()):.2f} of the tolerance"
            seen = (lim > 0)[:, None].expand(new, hq)
            assert not out[at:at + new][~seen].any()
        at += new


ATTEND = [
    # dtype, (new, held) of the sequences, Hq, Hkv, D, Dv, page, causal
    (torch.float16, [(1, 1)], 1, 1, 64, 64, 16, True),
    (torch.float16, [(1, 700)], 8, 8, 64, 64, 16, True),
    (torch.float16, [(1, 65), (1, 64), (1, 63), (1, 1), (1, 2049)], 8, 2, 128, 128, 32, True),
    (torch.float16, [(1, 513), (0, 77), (1, 0), (3, 2), (4, 4), (2, 300)], 6, 2, 128, 64, 64, True),   # rows that see nothing
    (torch.float16, [(7, 333), (5, 5), (1, 1000)], 12, 4, 80, 128, 16, True),
    (torch.float16, [(5, 333), (16, 90)], 4, 4, 8, 24, 256, False),
    (torch.float16, [(33, 200), (1, 3000), (64, 64), (20, 500)], 32, 8, 128, 128, 128, True),
    (torch.float16, [(150, 470), (257, 257), (1, 900)], 10, 2, 64, 64, 16, True),
    (torch.float16, [(300, 310)], 7, 1, 128, 128, 64, False),
    (torch.float16, [(2, 40)], 64, 1, 128, 128, 16, True),
    (torch.float16, [(300, 900), (129, 129), (5, 4000)], 16, 4, 128, 128, 16, True),
    (torch.float16, [(200, 513)], 8, 8, 96, 72, 32, True),
    (torch.float16, [(200, 150), (170, 0), (140, 129)], 4, 2, 64, 128, 64, True),                       # chunks past their cache
    (torch.float16, [(520, 1032), (0, 5), (300, 300)], 2, 1, 128, 64, 512, True),
    (torch.float16, [(70, 300)] * 40, 8, 8, 64, 64, 16, True),                                          # more items than SMs
    (torch.float16, [(3, 100), (40, 41), (0, 3), (1, 700)] * 10, 8, 1, 128, 64, 32, True),              # over 32 sequences of chunks
    (torch.float16, [(1, 1 + 37 * n % 500) for n in range(300)], 2, 1, 64, 64, 16, True),               # over 128 of single tokens
    (torch.float16, [(4, 20000)], 4, 1, 64, 64, 64, True),                                              # many pieces
    (torch.float16, [(1, 9000), (1, 5)], 33, 1, 64, 128, 128, True),                                    # wide groups
    (torch.float16, [(3, 40), (1, 500)], 128, 1, 128, 128, 16, True),
    (torch.float16, [(1, 50), (3, 400)], 130, 1, 64, 64, 16, True),
    (torch.float16, [(2, 90)], 260, 2, 128, 128, 16, False),
    (torch.float32, [(1, 1 + 53 * n % 300) for n in range(200)], 1, 1, 128, 128, 16, True),
    (torch.float32, [(2, 15000)], 8, 1, 128, 128, 32, True),
    (torch.float32, [(1, 1), (1, 130)], 2, 2, 64, 64, 16, True),
    (torch.float32, [(4, 333), (1, 2000), (2, 1), (0, 9), (3, 0)], 6, 2, 128, 128, 32, True),
    (torch.float32, [(40, 200), (7, 64)], 8, 4, 40, 96, 16, False),
    (torch.float32, [(130, 300), (1, 77)], 4, 1, 128, 64, 64, True),
    (torch.float32, [(257, 300)], 2, 2, 64, 64, 16, True),
    (torch.float32, [(5, 333), (1, 90), (2, 7)], 3, 1, 8, 24, 256, False),                              # tiles of 8 rows, part filled
    (torch.float32, [(3, 500), (1, 41), (0, 70)], 10, 2, 96, 72, 16, True),
    (torch.float32, [(1, 3000), (14, 60), (1, 2), (2, 1)], 1, 1, 64, 128, 64, True),
    (torch.float32, [(1, 40), (1, 0), (1, 1200)], 16, 1, 128, 64, 16, True),
]


@pytest.mark.parametrize("case", ATTEND)
def test_attend(case):
    dtype, lens, hq, hkv, d, dv, page, causal = case
    s = make(dtype, lens, hq, hkv, d, dv, page, seed=len(lens) + d)
    scale = d ** -0.5
    check_attend(s, lens, scale, causal, fa.paged_sdpa(**s, scale=scale, causal_mask=causal))
    assert fa.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("scale", [-0.3, 0.0, 4.0])
def test_scales_and_large_scores(dtype, scale):
    """Sharp, flat and negative scales; queries large enough for scores of several hundred."""
    lens = [(3, 200), (1, 70), (140, 260)]
    s = make(dtype, lens, 4, 2, 64, 64, 16, seed=5, amp=4.0 if dtype == torch.float16 else 1.0)
    check_attend(s, lens, scale, True, fa.paged_sdpa(**s, scale=scale))


def test_rows_behind_the_last_sequence_are_left():
    lens = [(2, 50), (140, 300)]
    for dtype in (torch.float16, torch.float32):
        s = make(dtype, lens, 4, 2, 64, 64, 16, tail=9)
        T = s["q"].shape[0]
        out, stats = torch.full((T, 4, 64), 7.0, dtype=dtype, device="cuda"), torch.full((T, 4), 7.0, device="cuda")
        got = fa.paged_sdpa(**s, scale=0.125, out=(out, stats))
        assert got[0] is out
        check_attend(s, lens, 0.125, True, got)
        assert (out[-9:] == 7).all() and (stats[-9:] == 7).all()
        k, v = torch.randn(T, 2, 64, device="cuda").to(dtype), torch.randn(T, 2, 64, device="cuda").to(dtype)
        before = s["k_pages"].clone(), s["v_pages"].clone()
        fa.paged_append(k, v, s["k_pages"], s["v_pages"], s["page_table"], s["kv_len"], s["q_start"])
        changed = (s["k_pages"] != before[0]) & ~(s["k_pages"].isnan() & before[0].isnan())
        assert int(changed.any(-1).any(-1).sum()) <= 142
        assert fa.device_status() == 0


def test_pages_and_lengths_out_of_range_stay_out_of_memory():
    """Bad page ids read as zeros, lengths past the table are clamped; both are reported."""
    for dtype, new in ((torch.float16, 1), (torch.float16, 200), (torch.float32, 2)):
        lens = [(new, 300), (new, 300)]
        s = make(dtype, lens, 4, 2, 64, 64, 16)
        fa.device_status()
        bad = dict(s, page_table=s["page_table"].clone())
        bad["page_table"][0, 3], bad["page_table"][0, 5] = -1, bad["k_pages"].shape[0]
        got = fa.paged_sdpa(**bad, scale=0.125)
        assert fa.device_status() == 2
        zero = dict(s, page_table=s["page_table"].clone(), k_pages=s["k_pages"].clone(), v_pages=s["v_pages"].clone())
        for i in (3, 5):
            zero["k_pages"][s["page_table"][0, i].item()] = 0
            zero["v_pages"][s["page_table"][0, i].item()] = 0
        check_attend(zero, lens, 0.125, True, got)
        s["page_table"][:, 19] = 0  # the entry behind the last page in use
        s["k_pages"].nan_to_num_(0), s["v_pages"].nan_to_num_(0)
        capacity = s["page_table"].shape[1] * 16
        full = dict(s, kv_len=torch.full_like(s["kv_len"], capacity))
        over = dict(s, kv_len=torch.tensor([capacity + 1, 2 ** 31 - 1], dtype=torch.int32, device="cuda"))
        ref = fa.paged_sdpa(**full, scale=0.125, causal_mask=False)
        assert fa.device_status() == 0
        got = fa.paged_sdpa(**over, scale=0.125, causal_mask=False)
        assert fa.device_status() == 2
        assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
        before = s["k_pages"].clone()
        k = torch.randn(2 * new, 2, 64, device="cuda").to(dtype)
        s["page_table"].fill_(-7)
        fa.paged_append(k, k, s["k_pages"], s["v_pages"], s["page_table"], s["kv_len"], s["q_start"])
        assert fa.device_status() == 2 and torch.equal(before, s["k_pages"])
        neg = torch.full_like(s["kv_len"], -5)
        fa.paged_append(k, k, s["k_pages"], s["v_pages"], s["page_table"], neg, s["q_start"])
        assert fa.device_status() == 2 and torch.equal(before, s["k_pages"])


APPEND = [
    # dtype, lens, Hq (0: no queries), Hkv, D, Dv, page, rot, interleaved, norm, weight dtype
    (torch.float16, [(1, 1)], 1, 1, 64, 64, 16, 64, False, True, torch.float16),
    (torch.float16, [(1, 17), (1, 900), (0, 3), (1, 32)], 32, 8, 128, 128, 32, 128, False, True, torch.float32),
    (torch.float16, [(130, 400), (1, 1), (33, 33)], 6, 2, 80, 24, 16, 16, True, True, torch.float16),
    (torch.float16, [(40, 90)] * 20, 0, 1, 8, 128, 64, 8, False, False, torch.float16),
    (torch.float16, [(5, 9)], 3, 3, 40, 40, 16, 0, False, True, torch.float32),
    (torch.float16, [(1, 300)] * 40, 4, 1, 128, 64, 128, 0, False, False, torch.float16),
    (torch.float32, [(17, 60), (3, 3)], 4, 2, 64, 128, 16, 32, True, True, torch.float32),
    (torch.float32, [(1, 2)] * 300, 2, 1, 128, 8, 16, 128, False, True, torch.float32),
]


@pytest.mark.parametrize("case", APPEND)
def test_append(case):
    """Values bit for bit, keys and queries as qk_norm_rope gives them bit for bit, nothing else touched."""
    dtype, lens, hq, hkv, d, dv, page, rot, inter, norm, wdt = case
    s = make(dtype, lens, max(hq, 1) * hkv, hkv, d, dv, page, seed=3)
    g = torch.Generator(device="cuda").manual_seed(9)
    T = s["q"].shape[0]
    k, v = torch.randn(T, hkv, d, generator=g, device="cuda").to(dtype), torch.randn(T, hkv, dv, generator=g, device="cuda").to(dtype)
    q = torch.randn(T, hq, d, generator=g, device="cuda").to(dtype) if hq else None
    qw, kw = ((1 + 0.1 * torch.randn(d, generator=g, device="cuda")).to(wdt) for _ in range(2)) if norm else (None, None)
    table = fa.rotary_table(1024, rot, device="cuda") if rot else None
    pos = torch.cat([torch.arange(h - a, h) for a, h in lens]).cuda()
    seq = torch.cat([torch.full((a,), n) for n, (a, _) in enumerate(lens)]).cuda()
    want_k, want_v = s["k_pages"].clone(), s["v_pages"].clone()
    where = (s["page_table"][seq, pos // page].long(), pos % page)
    qs = k if q is None else q
    rq, rk = fa.qk_norm_rope(qs, k, None if q is None else qw, kw, table, pos, pos, eps=1e-5, interleaved=inter)
    want_k[where], want_v[where] = rk, v
    got = fa.paged_append(k, v, s["k_pages"], s["v_pages"], s["page_table"], s["kv_len"], s["q_start"], q=q,
                          q_weight=None if q is None else qw, k_weight=kw, table=table, eps=1e-5, interleaved=inter)
    assert (got is None) if q is None else torch.equal(got, rq)
    for a, b in ((s["k_pages"], want_k), (s["v_pages"], want_v)):
        assert torch.equal(a.view(torch.int16 if dtype == torch.float16 else torch.int32),
                           b.view(torch.int16 if dtype == torch.float16 else torch.int32))
    assert fa.device_status() == 0


def test_append_reads_a_fused_projection_in_place():
    lens, H, D = [(5, 40), (1, 7)], 2, 64
    s = make(torch.float16, lens, H, H, D, D, 16)
    fused = torch.randn(6, 3 * H * D, device="cuda").half()
    q, k, v = (fused[:, i * H * D:(i + 1) * H * D].view(6, H, D) for i in range(3))
    table = fa.rotary_table(64, D, device="cuda")
    pools = [(s["k_pages"].clone(), s["v_pages"].clone()) for _ in range(2)]
    outs = [fa.paged_append(f(k), f(v), *pool, s["page_table"], s["kv_len"], s["q_start"], q=f(q), table=table)
            for f, pool in zip((lambda x: x, lambda x: x.contiguous()), pools)]
    assert torch.equal(*outs)
    assert torch.equal(pools[0][0].nan_to_num(3), pools[1][0].nan_to_num(3))
    assert torch.equal(pools[0][1].nan_to_num(3), pools[1][1].nan_to_num(3))
    a = fa.paged_sdpa(q, *pools[0], s["page_table"], s["kv_len"], s["q_start"])
    b = fa.paged_sdpa(q.contiguous(), *pools[0], s["page_table"], s["kv_len"], s["q_start"])
    assert torch.equal(a[0], b[0])


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_prompt_then_tokens_equals_one_causal_call(dtype):
    """A prompt in two chunks and then token by token, through norm, rotation, write and attention: the same
    rows as norm, rotation and causal sdpa over the whole sequence."""
    H, D, S, page = 4, 64, 300, 16
    g = torch.Generator(device="cuda").manual_seed(11)
    q, k, v = (torch.randn(2, S, H, D, generator=g, device="cuda").to(dtype) for _ in range(3))
    qw, kw = ((1 + 0.1 * torch.randn(D, generator=g, device="cuda")).to(dtype) for _ in range(2))
    table = fa.rotary_table(S, D, device="cuda")
    rq, rk = fa.qk_norm_rope(q, k, qw, kw, table)
    ref, ref_s = fa.sdpa_bshd(rq, rk, v, 0, 0, scale=D ** -0.5, causal_mask=True)
    pages = -(-S // page)
    k_pages = torch.full((2 * pages, page, H, D), float("nan"), dtype=dtype, device="cuda")
    v_pages = k_pages.clone()
    pt = torch.randperm(2 * pages, generator=torch.Generator().manual_seed(0)).int().view(2, pages).cuda()
    out, stats, at = torch.zeros_like(q), torch.zeros(2, H, S, device="cuda"), 0
    for step in [170, 125, 1, 1, 3]:
        x = [t[:, at:at + step].reshape(2 * step, H, D) for t in (q, k, v)]
        at += step
        kv_len = torch.full((2,), at, dtype=torch.int32, device="cuda")
        q_start = torch.tensor([0, step, 2 * step], dtype=torch.int32, device="cuda")
        qq = fa.paged_append(x[1], x[2], k_pages, v_pages, pt, kv_len, q_start, q=x[0], q_weight=qw, k_weight=kw, table=table)
        o, st = fa.paged_sdpa(qq, k_pages, v_pages, pt, kv_len, q_start, scale=D ** -0.5)
        out[:, at - step:at] = o.view(2, step, H, D)
        stats[:, :, at - step:at] = st.view(2, step, H).transpose(1, 2)
    assert fa.device_status() == 0
    # both sides are within the bounds of this file of the same values; |o| and A stay below 6 here
    u = HALF_STEP[dtype]
    tol = 2 * (2 * u * 6 + 300 * 2.0 ** -25 * 6 + 2.0 ** -13) if dtype == torch.float16 else 2 * 2.0 ** -16
    assert (out.double() - ref.double()).abs().max() <= tol
    assert (stats - ref_s).abs().max() <= 2.0 ** -13 if dtype == torch.float16 else 2.0 ** -15


def test_captured_step_follows_lengths_and_pages():
    """One captured append + attend step, replayed with other lengths, pages and a padded batch; two graphs and
    an eager call at once on three streams."""
    s = make(torch.float16, [(1, 704)] * 3, 8, 2, 128, 128, 16, seed=2, tail=1)
    s["page_table"] = torch.arange(132, dtype=torch.int32, device="cuda").view(3, 44)
    s["k_pages"].nan_to_num_(0), s["v_pages"].nan_to_num_(0)
    T = s["q"].shape[0]
    k, v = torch.randn(T, 2, 128, device="cuda").half(), torch.randn(T, 2, 128, device="cuda").half()
    table = fa.rotary_table(1024, 128, device="cuda")

    def step(pools):
        q = fa.paged_append(k, v, *pools, s["page_table"], s["kv_len"], s["q_start"], q=s["q"], table=table)
        return fa.paged_sdpa(q, *pools, s["page_table"], s["kv_len"], s["q_start"], scale=0.1)

    pools = [(s["k_pages"].clone(), s["v_pages"].clone()) for _ in range(3)]
    for pool in pools:  # (a write each: the three stay alike)
        step(pool)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for i in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(step(pools[i]))
        graphs.append(gr)
    for held in ([130, 40, 700], [1, 90, 64], [400, 1, 3]):
        s["kv_len"].copy_(torch.tensor(held, dtype=torch.int32))
        s["page_table"].copy_(torch.randperm(132).view(3, 44))
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in range(3)]
        with torch.cuda.stream(streams[0]):
            graphs[0].replay()
        with torch.cuda.stream(streams[1]):
            graphs[1].replay()
        with torch.cuda.stream(streams[2]):
            eager = step(pools[2])
        torch.cuda.synchronize()
        for o in outs:
            assert torch.equal(o[0][:3], eager[0][:3]) and torch.equal(o[1][:3], eager[1][:3])
        check_attend(dict(s, q=fa.qk_norm_rope(s["q"], s["q"], table=table, q_positions=torch.tensor(
            [h - 1 for h in held] + [0], device="cuda"))[0], k_pages=pools[2][0], v_pages=pools[2][1]),
            [(1, h) for h in held], 0.1, True, eager)
    assert fa.device_status() == 0


def test_offsets_past_32_bits():
    """Pages whose byte and element offsets do not fit 32 bits."""
    page, hkv, d = 256, 8, 128
    pool = (1 << 32) // (page * hkv * d) + 2  # elements past 2^32: 8.6 GB a pool
    k_pages = torch.empty(pool, page, hkv, d, dtype=torch.float16, device="cuda")
    v_pages = torch.empty(pool, page, hkv, d, dtype=torch.float16, device="cuda")
    far = torch.tensor([[pool - 1, pool - 2, 0]], dtype=torch.int32, device="cuda")
    lens = [(2, 600)]
    s = dict(page_table=far, kv_len=torch.tensor([600], dtype=torch.int32, device="cuda"),
             q_start=torch.tensor([0, 2], dtype=torch.int32, device="cuda"))
    big = dict(s, q_start=torch.tensor([0, 600], dtype=torch.int32, device="cuda"))
    k, v = (torch.randn(600, hkv, d, device="cuda").half() for _ in range(2))
    fa.paged_append(k, v, k_pages, v_pages, far, big["kv_len"], big["q_start"])
    assert torch.equal(k_pages[pool - 1], k[:256]) and torch.equal(v_pages[pool - 2], v[256:512]) and torch.equal(k_pages[0, :88], k[512:])
    for q_start, new in ((s["q_start"], 2), (big["q_start"], 600)):
        q = torch.randn(new, 16, d, device="cuda").half()
        got = fa.paged_sdpa(q, k_pages, v_pages, far, s["kv_len"], q_start, scale=d ** -0.5)
        check_attend(dict(s, q=q, k_pages=k_pages, v_pages=v_pages), [(new, 600)], d ** -0.5, True, got)
    assert fa.device_status() == 0


def test_host_mirror_refusals_on_the_device():
    s = make(torch.float16, [(1, 20)], 4, 2, 64, 64, 16)
    E = fa.InvalidArgumentError
    for change, words in [
        (dict(page_table=s["page_table"].long()), "page_table"), (dict(kv_len=s["kv_len"].cpu()), "CUDA tensors only"),
        (dict(q_start=s["q_start"][:1]), "page_table must be"), (dict(k_pages=s["k_pages"].transpose(1, 2)), "contiguous"),
        (dict(v_pages=s["v_pages"][:1]), "same pages"), (dict(k_pages=s["k_pages"].float()), "share dtype"),
        (dict(q=s["q"][:, :3]), "multiple of H_kv"), (dict(q=s["q"][..., :32]), "q must be"),
        (dict(k_pages=s["k_pages"][:, :8].contiguous(), v_pages=s["v_pages"][:, :8].contiguous()), "power of two"),
        (dict(out=(torch.empty(1, 4, 64, device="cuda"), torch.empty(1, 4, device="cuda"))), "out"),
    ]:
        with pytest.raises(E, match=words):
            fa.paged_sdpa(**{**s, **change})
    k = torch.zeros(1, 2, 64, device="cuda").half()
    rest = (s["k_pages"], s["v_pages"], s["page_table"], s["kv_len"], s["q_start"])
    w = torch.ones(64, device="cuda")
    for args, kw, words in [((k[:, :1], k, *rest), {}, "k must be"), ((k, k.float(), *rest), {}, "share dtype"),
                            ((k, k, *rest), dict(q_weight=w), "without q"), ((k, k, *rest), dict(k_weight=w[:32]), "weight"),
                            ((k, k, *rest), dict(k_weight=w.double()), "weights must"),
                            ((k, k, *rest), dict(table=torch.zeros(4, 72, device="cuda")), "rotary_dim"),
                            ((k, k, *rest), dict(q=k, q_weight=w, k_weight=w.half()), "share a dtype")]:
        with pytest.raises(E, match=words):
            fa.paged_append(*args, **kw)


def test_results_may_not_lie_over_the_queries():
    s = make(torch.float16, [(1, 20), (2, 9)], 4, 2, 64, 64, 16)
    pool = torch.zeros(6, 4, 64, device="cuda", dtype=torch.float16)
    s["q"] = pool[:3]
    stats = torch.empty(3, 4, device="cuda")
    for out in (pool[:3], pool[2:5]):
        with pytest.raises(fa.InvalidArgumentError, match="share memory"):
            fa.paged_sdpa(**s, out=(out, stats))
    with pytest.raises(fa.InvalidArgumentError, match="share memory"):
        fa.paged_sdpa(**s, out=(pool[3:], pool.view(torch.float32).view(-1)[:12].view(3, 4)))
    fa.paged_sdpa(**s, out=(pool[3:], stats))  # beside them


@pytest.mark.parametrize("dtype,new", [(torch.float16, 1), (torch.float16, 200), (torch.float32, 3)])
def test_a_nan_key_reaches_the_rows_that_see_it_and_no_others(dtype, new):
    lens = [(new, 300), (new, 250)]
    s = make(dtype, lens, 4, 2, 64, 64, 16, seed=4)
    clean = fa.paged_sdpa(**s, scale=0.125)
    for key in (297, 298, 299):  # of the first sequence, in the chunk's last columns or the token's own
        k_pages = s["k_pages"].clone()
        k_pages[s["page_table"][0, key // 16].item(), key % 16, 0] = float("nan")  # KV head 0: query heads 0 and 1
        got = fa.paged_sdpa(**dict(s, k_pages=k_pages), scale=0.125)
        sees = torch.zeros(2 * new, 4, dtype=torch.bool, device="cuda")
        sees[max(0, key - (300 - new)):new, :2] = True
        for a, b in zip(got, clean):
            seen = sees if a.dim() == 2 else sees[..., None].expand_as(a)
            assert a[seen].isnan().all() and torch.equal(a[~seen], b[~seen])
