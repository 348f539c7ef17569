"""Arguments of the beam operators that are refused on the host, before any GPU work."""
import pytest

from tests.test_i8_beam_refusals import at, err, select
from vkwr_amd import capi


@pytest.mark.parametrize("change,text", [
    ({"logits": at(9)}, "logits"), ({"logits": at(9) - 8}, "logits"), ({"ins": (at(9) + 16, at(2), at(3))}, "input"),
    ({"ins": (at(1), at(9) - 4, at(3))}, "input"), ({"ins": (at(1), at(2), at(9))}, "input")])
def test_select_refuses_a_workspace_over_its_inputs(change, text):
    assert select(**change) == 1 and "workspace" in err() and text in err()


def test_select_looks_at_the_used_part_of_the_workspace_only():
    """Inputs may lie in the same buffer, behind what the call needs."""
    need = capi.beam_workspace_bytes(2, 3, 8)
    assert select(logits=at(9) + need - 4) == 1 and "workspace" in err()
    assert select(logits=at(9) + need, alpha=-1.0) == 1 and "length penalty" in err()
