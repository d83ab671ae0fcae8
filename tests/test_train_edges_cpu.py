"""The training operators' Python entry points without a GPU."""
import pytest

from tests.conftest import load_samrs


def test_a_repeated_bad_shape_reports_its_own_error():
    """The message belongs to the call, whatever failed in between."""
    s = load_samrs()

    def refusal():
        with pytest.raises(s.SamrsError) as e:
            s._workspace(s._bwd_workspace_bytes(1, 4, 4, 129, 0), "cpu")
        return e.value.code, str(e.value)

    first = refusal()
    assert first[0] == s._abi.ERR_UNSUPPORTED and "head_dim 129" in first[1]
    assert s._abi.lib().samrs_layer_norm_bwd_workspace(-1, 8) == s._abi.ERR_INVALID
    assert refusal() == first
    s._abi.lib().samrs_layer_norm_bwd_workspace(1, 8)  # a call that succeeds clears the last message
    assert refusal() == first
