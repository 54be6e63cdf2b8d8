"""Refusals of the rotary and paged operators that need no GPU: the C ABI's argument checks and the host mirror's."""
import importlib

import pytest

torch = pytest.importorskip("torch")

fa = importlib.import_module("tf-custom-flash-attention_b200")
L = fa._lib.lib()
EINVAL, EUNSUPPORTED, EWORKSPACE = fa._lib.EINVAL, fa._lib.EUNSUPPORTED, fa._lib.EWORKSPACE
A = 4096  # an aligned address that no refused call may touch


def rope(dtype=0, q=A, q_tokens=4, q_heads=2, q_stride=128, q_positions=None, q_period=4, k=A, k_tokens=4, k_heads=1,
         k_stride=64, k_positions=None, k_period=4, D=64, q_weight=A, k_weight=A, weight_dtype=0, eps=1e-6, table=A,
         max_positions=8, rotary_dim=64, interleaved=0, q_out=A, k_out=A):
    return L.sdpa_b200_qk_norm_rope(dtype, q, q_tokens, q_heads, q_stride, q_positions, q_period, k, k_tokens, k_heads,
                                    k_stride, k_positions, k_period, D, q_weight, k_weight, weight_dtype, eps, table,
                                    max_positions, rotary_dim, interleaved, q_out, k_out, None)


@pytest.mark.parametrize("change,code", [
    (dict(dtype=2), EINVAL), (dict(D=60), EINVAL), (dict(D=0), EINVAL), (dict(D=136, q_stride=272, k_stride=136), EUNSUPPORTED),
    (dict(rotary_dim=72), EINVAL), (dict(rotary_dim=12), EINVAL), (dict(rotary_dim=-8), EINVAL), (dict(table=None), EINVAL),
    (dict(table=A + 4), EINVAL), (dict(max_positions=0), EINVAL), (dict(max_positions=1 << 31), EINVAL),
    (dict(weight_dtype=7), EINVAL), (dict(dtype=1, weight_dtype=0), EINVAL), (dict(q=None), EINVAL), (dict(q=A + 2), EINVAL),
    (dict(q_out=None), EINVAL), (dict(k_out=A + 8), EINVAL), (dict(q_stride=64), EINVAL), (dict(q_stride=132), EINVAL),
    (dict(q_tokens=-1), EINVAL), (dict(q_tokens=1 << 31), EINVAL), (dict(k_heads=70000), EINVAL), (dict(q_period=0), EINVAL),
    (dict(q_tokens=0, k_heads=0), 0),
])
def test_rope_abi_refusals(change, code):
    assert rope(**change) == code


def rope_bwd(dq_out=A, dk_out=A, dqw=A, dkw=A, qw=A, kw=A, ws=A, ws_bytes=1 << 24, stride=128, tokens=4):
    return L.sdpa_b200_qk_norm_rope_bwd(0, A, dq_out, tokens, 2, 128, stride, None, 4, A, dk_out, tokens, 2, 128, 128, None,
                                        4, 64, qw, kw, 0, 1e-6, A, 8, 64, 0, A, A, dqw, dkw, ws, ws_bytes, None)


@pytest.mark.parametrize("change,code", [
    (dict(dq_out=None), EINVAL), (dict(dk_out=A + 4), EINVAL), (dict(dqw=None), EINVAL), (dict(kw=None), EINVAL),
    (dict(stride=120), EINVAL), (dict(ws=None), EWORKSPACE), (dict(ws_bytes=1000), EWORKSPACE), (dict(ws=A + 2), EWORKSPACE),
])
def test_rope_bwd_abi_refusals(change, code):
    assert rope_bwd(**change) == code


def append(dtype=0, q=A, q_stride=256, k=A, k_stride=128, v=A, v_stride=128, tokens=4, H_q=4, H_kv=2, D=64, D_v=64,
           q_out=A, k_pages=A, v_pages=A, num_pages=9, page=16, pt=A, width=3, kv_len=A, q_start=A, seqs=2):
    return L.sdpa_b200_paged_append(dtype, q, q_stride, k, k_stride, v, v_stride, tokens, H_q, H_kv, D, D_v, None, None, 0,
                                    1e-6, None, 0, 0, 0, q_out, k_pages, v_pages, num_pages, page, pt, width, kv_len,
                                    q_start, seqs, None)


def attend(dtype=0, q=A, q_stride=256, k_pages=A, v_pages=A, out=A, stats=A, tokens=4, H_q=4, H_kv=2, D=64, D_v=64,
           num_pages=9, page=16, pt=A, width=3, kv_len=A, q_start=A, seqs=2, ws=A, ws_bytes=1 << 30):
    return L.sdpa_b200_paged_sdpa(dtype, q, q_stride, k_pages, v_pages, out, stats, tokens, H_q, H_kv, D, D_v, num_pages,
                                  page, pt, width, kv_len, q_start, seqs, 0.125, 1, ws, ws_bytes, None)


BOTH = [
    (dict(dtype=3), EINVAL), (dict(D=12), EINVAL), (dict(D_v=4), EINVAL), (dict(page=8), EINVAL), (dict(page=48), EINVAL),
    (dict(page=131072), EINVAL), (dict(width=1 << 28), EINVAL), (dict(width=-1), EINVAL), (dict(num_pages=1 << 31), EINVAL),
    (dict(pt=None), EINVAL), (dict(kv_len=None), EINVAL), (dict(q_start=None), EINVAL), (dict(k_pages=None), EINVAL),
    (dict(v_pages=A + 8), EINVAL), (dict(q_stride=100), EINVAL), (dict(q=A + 4), EINVAL), (dict(seqs=1 << 31), EINVAL),
    (dict(tokens=-1), EINVAL), (dict(tokens=0), 0), (dict(seqs=0), 0),
]


@pytest.mark.parametrize("change,code", BOTH + [(dict(H_kv=0), EINVAL), (dict(D_v=200, v_stride=400), EUNSUPPORTED),
                                                (dict(k=None), EINVAL), (dict(v_stride=64), EINVAL), (dict(q_out=None), EINVAL)])
def test_append_abi_refusals(change, code):
    assert append(**change) == code


@pytest.mark.parametrize("change,code", BOTH + [(dict(H_q=5), EINVAL), (dict(H_q=1), EINVAL), (dict(D=136, q_stride=544), EUNSUPPORTED),
                                                (dict(out=None), EINVAL), (dict(stats=None), EINVAL), (dict(tokens=1 << 30), EINVAL),
                                                (dict(ws=None), EWORKSPACE), (dict(ws=A + 4), EWORKSPACE), (dict(ws_bytes=64), EWORKSPACE)])
def test_attend_abi_refusals(change, code):
    assert attend(**change) == code


def test_host_mirror_refusals():
    x = torch.zeros(2, 4, 3, 64)
    E = fa.InvalidArgumentError
    with pytest.raises(E, match="CUDA tensors only"):
        fa.qk_norm_rope(x, x)
    with pytest.raises(E, match="rank 2"):
        fa.qk_norm_rope(x[0, 0], x)
    with pytest.raises(E, match="K feature size mismatch"):
        fa.qk_norm_rope(x, x[..., :32])
    with pytest.raises(E, match="multiple of 8"):
        fa.qk_norm_rope(x[..., :60], x[..., :60])
    with pytest.raises(E, match="feature size over 128"):
        fa.qk_norm_rope(torch.zeros(1, 1, 1, 136), torch.zeros(1, 1, 1, 136))
    with pytest.raises(E, match="half or float"):
        fa.qk_norm_rope(x.double(), x.double())
    with pytest.raises(E, match="share dtype"):
        fa.qk_norm_rope(x, x.half())
    for bad in (12, 0, -8):
        with pytest.raises(E, match="rotary_dim"):
            fa.rotary_table(4, bad, device="cpu")
    with pytest.raises(E, match="max_positions"):
        fa.rotary_table(0, 8, device="cpu")
    i = torch.zeros(2, dtype=torch.int32)
    pool = torch.zeros(4, 16, 2, 64)
    with pytest.raises(E, match="CUDA tensors only"):
        fa.paged_sdpa(x[0], pool, pool, i.view(1, 2), i[:1], i)
    with pytest.raises(E, match="CUDA tensors only"):
        fa.paged_append(x[0], x[0], pool, pool, i.view(1, 2), i[:1], i)
    with pytest.raises(E, match="rank"):
        fa.paged_sdpa(x, pool, pool, i.view(1, 2), i[:1], i)


def test_rotary_table_values():
    t = fa.rotary_table(70, 16, base=500.0, device="cpu")
    assert t.shape == (70, 16) and t.dtype == torch.float32
    ang = 69 * 500.0 ** (-torch.arange(0, 16, 2, dtype=torch.float64) / 16)
    ref = torch.cat([ang.cos(), ang.sin()])
    assert (t[69].double() - ref).abs().max() <= 2.0 ** -25 + 1e-15


def test_workspace_queries():
    assert L.sdpa_b200_paged_workspace_bytes(0, 0, 1, 1, 1, 64, 64) == 0
    assert L.sdpa_b200_paged_workspace_bytes(0, 4, 4, 8, 2, 64, 64) > 0
    assert L.sdpa_b200_qk_norm_rope_bwd_workspace_bytes(0) == 0
    assert L.sdpa_b200_qk_norm_rope_bwd_workspace_bytes(64) == 592 * 2 * 64 * 4


@pytest.mark.parametrize("change", [dict(page_size=48), dict(page_size=8), dict(head_dim=12), dict(head_dim=136),
                                    dict(value_dim=4), dict(pages=0), dict(heads=0), dict(dtype=torch.bfloat16)])
def test_cache_refusals(change):
    with pytest.raises(fa.InvalidArgumentError):
        fa.PagedCache(**{**dict(pages=4, page_size=16, heads=2, head_dim=64, device="cpu"), **change})


def test_shared_memory_is_seen():
    x = torch.empty(64)
    share = importlib.import_module("tf-custom-flash-attention_b200.paged")._share_bytes
    assert share(x[:8], x[7:]) and share(x[::4], x[1:2]) and share(x, x)
    assert not share(x[:8], x[8:]) and not share(x[:0], x) and not share(x[0:8:2], x[7:])
