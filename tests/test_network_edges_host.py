"""The attribute network on the host, where its parts meet: what is passed on and what is refused, without a GPU."""
import pytest


def test_only_muon_takes_copies():
    from tinygs_amd.optim import create_optimizer
    with pytest.raises(RuntimeError, match="writes no copies"):
        create_optimizer("simple_adam", None, None, copies=[])
