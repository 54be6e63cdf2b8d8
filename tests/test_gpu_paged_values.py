"""paged_sdpa in float: values of any magnitude (needs a B200).

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
