"""What the serving layer and its operators refuse or follow: positions past the rotation table, changed arguments."""
import importlib

import pytest

torch = pytest.importorskip("torch")

fa = importlib.import_module("tf-custom-flash-attention_b200")


def test_a_batch_knows_its_longest_sequence():
    c = fa.PagedCache(8, 16, 2, 8, device="cpu")
    assert c.batch([("a", 17), ("b", 3)]).longest == 17
    assert c.batch([("b", 2)]).longest == 5
    assert c.batch([("b", 1), ("a", 0)]).longest == 6  # ("a" has no new tokens)
    assert c.batch([]).longest == 0
    b = c.batch([("a", 1)])
    assert fa.PagedBatch(b.page_table, b.kv_len, b.q_start, b.tokens).longest is None  # (lengths on the device alone)


def test_paged_layer_refuses_positions_past_its_table():
    """The same mistake as in forward, and the same error, before anything is written to the cache."""
    m = fa.MHA(num_heads=2, rotary_dim=8, max_positions=20).eval()
    c = fa.PagedCache(8, 16, 2, 8, device="cpu")
    x = torch.zeros(1, 16)
    c.batch([("a", 20)])
    batch = c.batch([("a", 1)])
    with pytest.raises(ValueError, match="21 tokens with max_positions 20"):
        m.forward_paged(x, x, x, c, batch)
    assert not c.k_pages.any() and not c.v_pages.any()
    import types
    m._table = lambda device: None
    bare = types.SimpleNamespace(page_table=batch.page_table, kv_len=batch.kv_len, q_start=batch.q_start)
    with pytest.raises(fa.InvalidArgumentError, match="CUDA tensors only"):  # (as far as the write, where nothing is known)
        m.forward_paged(x, x, x, c, bare)
    plain = fa.MHA(num_heads=2).eval()  # without a rotation there is no table to leave
    with pytest.raises(fa.InvalidArgumentError, match="CUDA tensors only"):
        plain.forward_paged(x, x, x, c, batch)


@pytest.mark.gpu
def test_paged_layer_takes_the_last_position_of_its_table():
    m = fa.MHA(num_heads=2, rotary_dim=8, max_positions=20).cuda().eval()
    c = fa.PagedCache(8, 16, 2, 8)
    x = torch.randn(20, 16, device="cuda").half()
    assert m.forward_paged(x, x, x, c, c.batch([("a", 20)])).shape == x.shape
    batch = c.batch([("a", 1)])
    before = c.k_pages.clone()
    with pytest.raises(ValueError, match="max_positions"):
        m.forward_paged(x[:1], x[:1], x[:1], c, batch)
    assert torch.equal(before, c.k_pages) and fa.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("change", [dict(max_positions=64), dict(rotary_base=100.0), dict(rotary_dim=16)])
def test_the_rotation_follows_changed_attributes(change):
    kw = dict(num_heads=2, rotary_dim=32, max_positions=16)
    m = fa.MHA(**kw).cuda().eval()
    x = torch.randn(1, 16, 64, device="cuda").half()
    m(x, x, x)  # (lays its table out)
    for name, value in change.items():
        setattr(m, name, value)
    new = fa.MHA(**{**kw, **change}).cuda().eval()
    y = torch.randn(1, new.max_positions, 64, device="cuda").half()
    assert torch.equal(m(y, y, y), new(y, y, y))
    assert fa.device_status() == 0


@pytest.mark.gpu
def test_results_may_not_lie_over_any_input_or_each_other():
    mem = torch.zeros(1 << 16, device="cuda", dtype=torch.float16)
    q, k_pages, v_pages = mem[:512].view(2, 4, 64), mem[4096:4096 + 4096].view(2, 16, 2, 64), mem[8192:8192 + 4096].view(2, 16, 2, 64)
    i32 = mem[16384:16384 + 64].view(torch.int32)
    i32.copy_(torch.tensor([0, 1, 2] + [0, 1] + [5, 9] + [0] * 25, dtype=torch.int32))
    q_start, page_table, kv_len = i32[:3], i32[3:5].view(2, 1), i32[5:7]
    args = (q, k_pages, v_pages, page_table, kv_len, q_start)
    out, stats = torch.empty(2, 4, 64, device="cuda", dtype=torch.float16), torch.empty(2, 4, device="cuda")
    lie = lambda at, n: mem[at:at + n]
    for at, name in ((0, "q"), (8184, "k_pages"), (8192 + 4088, "v_pages"), (16384, "q_start|kv_len|page_table")):
        with pytest.raises(fa.InvalidArgumentError, match=rf"out\[0\] must not share memory with ({name})"):
            fa.paged_sdpa(*args, out=(lie(at, 512).view(2, 4, 64), stats))
        with pytest.raises(fa.InvalidArgumentError, match=rf"out\[1\] must not share memory with ({name})"):
            fa.paged_sdpa(*args, out=(out, lie(at, 16).view(torch.float32).view(2, 4)))
    with pytest.raises(fa.InvalidArgumentError, match="out.0. and out.1."):
        fa.paged_sdpa(*args, out=(lie(20000, 512).view(2, 4, 64), lie(20504, 16).view(torch.float32).view(2, 4)))
    got = fa.paged_sdpa(*args, out=(lie(512, 512).view(2, 4, 64), lie(1024, 16).view(torch.float32).view(2, 4)))  # between them
    want = fa.paged_sdpa(*args)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and fa.device_status() == 0
