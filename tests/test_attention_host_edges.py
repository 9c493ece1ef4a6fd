"""Host side of rotary positions, the paged cache and attention at its edges (no GPU); beside test_attention_host.py."""
import numpy as np
import pytest

import ojas_engine_b200 as ob


@pytest.mark.parametrize("kw", [dict(factor=5e-324), dict(factor=1e-308, freq_factors=[1e-3] * 32)])
def test_frequencies_beyond_a_double_are_refused(kw):
    with pytest.raises(ob.OjasB200Error, match="frequenc"):
        ob.rope_frequencies(64, **kw)


def test_a_factor_that_no_pair_is_divided_by():
    """By parts, every pair turns more than beta_fast times (the slowest 4096 * 0.13 / 2 pi = 87): all keep their frequency, however
    far the divided one would lie beyond a double."""
    got = ob.rope_frequencies(64, factor=1e-308, freq_factors=[1e-3] * 32, orig_len=4096)
    assert np.allclose(got, ob.rope_frequencies(64, freq_factors=[1e-3] * 32), rtol=1e-15, atol=0)
