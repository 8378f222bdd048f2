"""How much work one call of attention over the paged cache takes: the host's check that 32 bits count it, at its border.  On
the host model, which has compute units to plan for without a device; no call here gets as far as a launch."""
import pytest

from tests.hostmodel.model import in_child
from tests.test_paged_refusals import _Args, _placed


@pytest.mark.parametrize("tokens,query_len,width", [
    # many rows: (2^25 / 256 + 2) tiles of 2 heads, so 0xFF000000 / 262148 = 16319 steps each, one for a page of 64 and two more
    (1 << 24, 0, 16317),
    # few rows, four to a tile: (2^17 / 4 + 2) tiles of 2 heads, so 0xFF000000 / 65540 = 65276 units of two pages, and two more
    (1 << 16, 1, 2 * 65274 + 1)])
@in_child
def test_more_work_than_a_list_counts_is_refused_at_the_border(tokens, query_len, width):
    from tests.hostmodel import build
    from tests.hostmodel.model import Model

    lib = Model(cus=256, lib_path=build.build()).lib
    for w, said in ((width, b"workspace"), (width + 1, b"several")):
        a = _Args()
        a.q, a.out = _placed(0), _placed(1 << 40)
        a.batch.num_tokens, a.batch.table_width, a.batch.table_stride = tokens, w, w
        a.max_query_len, a.workspace = query_len, None
        assert a.attend(lib) != 0
        assert said in lib.ci_last_error(), lib.ci_last_error()
