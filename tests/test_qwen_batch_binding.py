"""QwenDecoder.generate_batch hands the library a bound that it can refuse.  CPU."""
import numpy as np
import pytest


@pytest.mark.parametrize("maximum", [-1, 0, 1025, 2 ** 31, 2 ** 32, 2 ** 32 + 4, 2 ** 40])
def test_a_bound_out_of_range_is_refused_not_wrapped(gpt_mod, maximum):
    """2^32 + 4 is 4 to a C uint32: rows of ids would be 4 apart in the library and 2^32 + 4 in the result."""
    handed = []

    class Library:
        @staticmethod
        def itts_qwen_generate_batch(handle, n, ids, sizes, bound, *rest):
            handed.append(bound)
            return gpt_mod.ERR_INVALID_ARGUMENT

        @staticmethod
        def itts_qwen_last_error(handle):
            return b"Qwen generation capacity exceeded"

        @staticmethod
        def itts_qwen_destroy(handle):
            pass

    decoder = gpt_mod.QwenDecoder.__new__(gpt_mod.QwenDecoder)
    decoder._lib, decoder._h = Library, 1
    with pytest.raises(ValueError, match="capacity exceeded"):
        decoder.generate_batch([np.array([1, 2], np.uint32)] * 3, maximum)
    assert handed == [0]
