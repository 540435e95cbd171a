"""The ranges of the clear operators' numbers, in Python and at the C ABI (no GPU needed: what is refused launches
nothing, and a call without rows is looked at and launches nothing either)."""
import math

import pytest

import pfa_native as P
import pyPhantom as ph
from test_clear_ops import _abi, fake


@pytest.mark.parametrize("eps", [math.inf, -math.inf, math.nan, -1e-30])
def test_eps_refused(eps):
    """In Python, by what is wrong with it, and by the ABI."""
    with pytest.raises(ValueError, match="eps must be finite and 0 or more"):
        ph.rms_norm_int8(fake(2, 3), fake(3), eps)
    rc, said = _abi("pfa_rms_norm_int8", None, 0, None, 0, None, 0, 0, 8, eps, None, 0, None, 0, None, None)
    assert rc == P.PFA_ERR_INVALID_ARGUMENT and "eps must be finite and 0 or more" in said


@pytest.mark.parametrize("eps", [0.0, 1e-300, 1e31, 1e300])
def test_eps_taken(eps):
    assert _abi("pfa_rms_norm_int8", None, 0, None, 0, None, 0, 0, 8, eps, None, 0, None, 0, None, None)[0] == P.PFA_OK


@pytest.mark.parametrize("heat", [math.inf, math.nan, -1e-30])
def test_temperature_refused(heat):
    with pytest.raises(ValueError, match="temperature must be finite and 0 or more"):
        ph.token_probabilities(fake(2, 3), heat)


@pytest.mark.parametrize("heat,rc", [(0.0, P.PFA_OK), (1e31, P.PFA_OK), (3e38, P.PFA_OK), (math.inf, P.PFA_OK),
                                     (math.nan, P.PFA_ERR_INVALID_ARGUMENT), (-1.0, P.PFA_ERR_INVALID_ARGUMENT)])
def test_temperature_at_the_abi(heat, rc):
    """What a row's own temperature may be, one for all rows may be."""
    assert _abi("pfa_token_probabilities", None, 0, 0, 0, 5, None, heat, None, 0, None, None, 0, None)[0] == rc
