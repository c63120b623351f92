"""GatedExperts' choice of weights where the caller makes none: those of one expert a token are not brought to one, which would leave
the router without a gradient."""
from flashmlp_amd import GatedExperts


def test_weights_of_the_module():
    def normalize(k, **kw):
        return GatedExperts(4, 32, 40, k, device="cpu", **kw).normalize

    assert normalize(1) is False and normalize(2) is True and normalize(4) is True
    for k in (1, 2):
        for value in (True, False):
            assert normalize(k, normalize=value) is value
