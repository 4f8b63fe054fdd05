"""Every path that writes codes, with each code held to the nearest one: the tests of rows and of the cache in use, over
again, with the stricter check in place."""

import pytest

from tests import quant_util as Q
from tests import test_gpu_quant_rows as rows
from tests import test_gpu_quant_used as used
from tests.quant_nearest import assert_nearest


def cases(function):
    (mark,) = [m for m in function.pytestmark if m.name == "parametrize"]
    return [(function, dict(zip(mark.args[0].split(","), v if isinstance(v, tuple) and "," in mark.args[0] else (v,)))) for v in mark.args[1]]


CASES = [c for f in (rows.test_store, rows.test_store_of_unusual_rows, rows.test_copy_shifted, used.test_recorded_decode_steps,
                     used.test_decodes_and_chunks_in_one_step, used.test_blocks_are_merged_and_read) for c in cases(f)]
CASES = [(f, a) for f, a in CASES if not (f is rows.test_copy_shifted and (a["shift"] == 0 or a["rotary"] == 0))]  # (codes as they are)
CASES += [(rows.test_store_without_rotation_alignment_or_room, {}), (used.test_tensors_of_another_stream, {})]


@pytest.mark.gpu
@pytest.mark.parametrize("function,arguments", CASES, ids=lambda x: x.__name__ if callable(x) else "-".join(map(str, x.values())).replace(" ", ""))
def test_codes_are_the_nearest_ones(function, arguments, monkeypatch):
    seen = []
    monkeypatch.setattr(Q, "assert_quantises", lambda *a: (seen.append(1), assert_nearest(*a)))
    function(**arguments)
    assert seen
