"""Layers and routers: arguments that contradict one another are refused before
anything touches a GPU."""
import pytest


@pytest.mark.parametrize("t", [39, 2])
def test_norm_w_of_the_layer_and_of_its_router(pkg, t):
    """A layer asked to normalise with a router that does not would drop the wish without a word."""
    types = {r: t for r in ("gate", "up", "down")}
    with pytest.raises(pkg.MoeError, match="norm_w"):
        pkg.MoELayer(64, 64, 4, 2, types, norm_w=True, router=pkg.Router(2))
    with pytest.raises(pkg.MoeError, match="another number"):
        pkg.MoELayer(64, 64, 4, 2, types, norm_w=True, router=pkg.Router(3, norm_w=True))
