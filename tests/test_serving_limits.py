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
