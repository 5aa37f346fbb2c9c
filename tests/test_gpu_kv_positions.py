"""The rotation of appended rows (mit2cfm_kv_append_device) at every 32-bit position."""
from __future__ import annotations

import numpy as np
import pytest

pytest.importorskip("torch")

from ops_ref import Batch  # noqa: E402
from test_gpu_kv_ops import _append_check, ctx  # noqa: E402, F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("interleaved", [False, True])
def test_the_lowest_position_is_a_position(mit2, ctx, dtype, interleaved):  # noqa: F811
    b = Batch([5], [9], dim=64, dtype=dtype, seed=2)
    _append_check(mit2, ctx, b, 64, interleaved, position=np.array([-2 ** 31, -2 ** 31 + 1, 0, 2 ** 31 - 1, -2 ** 31], np.int32))
