"""What kvsnap_amd.attention refuses at its edges, without a GPU."""
import pytest

torch = pytest.importorskip("torch")
import torch.autograd.forward_ad as forward_ad

from kvsnap_amd.attention import PagedCache, rotate
from test_attention_host import ON_CPU, append, attend, built, layer, step  # noqa: F401  (built: a fixture)


@pytest.mark.parametrize("name", ["query", "key", "value", "query_out"])
def test_a_forward_mode_tangent_is_refused_not_dropped(name):
    given = step()
    given.setdefault("query_out", torch.zeros_like(given["query"]))
    with forward_ad.dual_level():
        given[name] = forward_ad.make_dual(given[name], torch.ones_like(given[name]))
        with pytest.raises(ValueError, match=f"^{name} carries a forward-mode tangent"):
            append(layer(), given)
        with torch.no_grad(), pytest.raises(ValueError, match="forward-mode tangent"):
            append(layer(), given)
        with torch.inference_mode(), pytest.raises(ValueError, match=ON_CPU):       # which turns both modes off
            append(layer(), given)
        if name == "query":
            given.pop("query_out")
            with pytest.raises(ValueError, match="query carries a forward-mode tangent"):
                attend(layer(), given)
        x = forward_ad.make_dual(torch.zeros((3, 2, 64)), torch.ones((3, 2, 64)))
        with pytest.raises(ValueError, match="x carries a forward-mode tangent"):
            rotate(x, torch.zeros(3, dtype=torch.int64), torch.zeros((5, 32, 2)))


def test_a_gradient_of_the_cache_or_of_the_table_is_refused_not_dropped():
    cache = torch.zeros((2, 4, 16, 2, 64), dtype=torch.bfloat16, requires_grad=True)
    learned = torch.zeros((5, 32, 2), requires_grad=True)
    for call in (append, attend):
        with pytest.raises(ValueError, match="the cache requires a gradient"):
            call(PagedCache(cache, 16), step())
        with torch.no_grad(), pytest.raises(ValueError, match=ON_CPU):
            call(PagedCache(cache, 16), step())
    for call in (lambda: append(layer(), step(), rotary=learned),
                 lambda: rotate(torch.zeros((3, 2, 64)), torch.zeros(3, dtype=torch.int64), learned)):
        with pytest.raises(ValueError, match="a rotary table requires a gradient"):
            call()
        with torch.no_grad(), pytest.raises(ValueError, match=ON_CPU):
            call()
