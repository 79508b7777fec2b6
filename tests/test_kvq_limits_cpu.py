"""The largest counts that the quantised-cache attention takes, and those above, refused before anything is launched: its
kernels count rows and runs in 32 bits and step past the last one."""
import pytest

from bitnetrs_b200 import InvalidShape
from test_kvq_cpu import attend, pages, prompt


@pytest.mark.parametrize("call", [attend, prompt])
def test_rows_that_32_bits_cannot_step_past(call):
    for rows in ((1 << 31) - 1, (1 << 31) - 600, (1 << 31) - 1024):
        with pytest.raises(InvalidShape) as e:
            call(pages(), rows=rows)
        assert "rows below" in e.value.expected
    with pytest.raises(InvalidShape) as e:
        call(pages(), rows=(1 << 31) - 1025)
    assert e.value.expected == "non-null context"


def test_runs_that_32_bits_cannot_search():
    for n in ((1 << 31) - 1, 1 << 30):
        with pytest.raises(InvalidShape) as e:
            prompt(pages(), n=n)
        assert "n_seqs below" in e.value.expected
    with pytest.raises(InvalidShape) as e:
        prompt(pages(), n=(1 << 30) - 1)
    assert e.value.expected == "non-null context"
