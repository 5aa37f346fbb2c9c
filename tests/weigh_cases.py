"""Sizes at which the attention weights' waves share their keys and divide the queries (kv_plan.h), for test_gpu_kv_weigh_queries.py, and what
test_weigh_plan.py holds them to: what a batch is made of (ops_ref.Batch), and whether its blocks go by XCDs."""
from __future__ import annotations


def case(new, before, *, dim, heads, dtype, page=16, by_xcd=False, **more):
    """A batch's arguments: new[s] rows after before[s] cached ones."""
    return dict(args=dict(new=list(new), length=[n + o for n, o in zip(new, before)], page=page, q_heads=heads[0], kv_heads=heads[1], dim=dim, dtype=dtype, **more),
                by_xcd=by_xcd)


# Every type and head size: through LDS (rows of up to 256 bytes, sizes that are powers of two) and straight into operands.
SIZES = [case([131, 0, 200], [300, 50, 3], dim=dim, heads=heads, dtype=dtype, lead_rows=2, tail_rows=1)
         for dtype in ("f32", "f16", "bf16") for dim, heads in ((32, (6, 2)), (64, (3, 3)), (96, (2, 1)), (128, (5, 1)), (192, (2, 1)), (256, (4, 2)))]
BIRTHS = [case([100, 0, 120], [90, 10, 1], dim=64, heads=(4, 2), dtype="f16", lead_rows=2, tail_rows=1),
          case([180, 3], [0, 200], dim=96, heads=(2, 2), dtype="f32", lead_rows=1),
          case([90, 110], [17, 300], dim=128, heads=(4, 4), dtype="bf16", by_xcd=True)]
# A weight's stride that cuts the lines short is a plan's length too.
STRIDES = [(stride, case([1, 160], [130, 50], dim=dim, heads=(4, 2), dtype=dtype)) for stride in (1, 63, 64, 65, 100, 300) for dim, dtype in ((64, "bf16"), (96, "f16"))]
# Lines by XCDs: eights of them, and with some blocks of the grid left over.
XCD = [case([(37 * s) % 61 + 30 for s in range(9)], [(29 * s) % 300 for s in range(9)], dim=64, heads=(16, 4), dtype="f16", page=8, by_xcd=True),
       case([(41 * s) % 50 + 40 for s in range(11)], [(31 * s) % 90 for s in range(11)], dim=96, heads=(12, 3), dtype="f32", by_xcd=True),
       case([60, 0, 90, 70], [200, 30, 0, 7], dim=32, heads=(8, 2), dtype="bf16", page=64, by_xcd=True),
       case([130] * 35, [5 * s for s in range(35)], dim=64, heads=(1, 1), dtype="bf16", by_xcd=True)]
LONG = case([150, 60], [2000, 70], dim=64, heads=(2, 2), dtype="bf16")
OTHERS = dict(in_place=case([100, 0, 90], [100, 7, 90], dim=64, heads=(2, 1), dtype="f32", page=8), odd_places=case([130, 90, 60], [100, 7, 0], dim=64, heads=(2, 1), dtype="f16"),
              unseen=case([110, 90], [0, 60], dim=64, heads=(2, 2), dtype="f32"), large=case([130, 4, 120], [300, 90, 60], dim=64, heads=(2, 1), dtype="f16"),
              last=case([300, 3, 0, 260], [240, 1, 8, 1], dim=64, heads=(4, 2), dtype="bf16", page=32, lead_rows=1, by_xcd=True))
LAST = 70  # rows that are counted of `last`
FINITE = [case([130, 90], [90, 40], dim=dim, heads=(2, 1), dtype=dtype) for dim, dtype in ((64, "f32"), (128, "bf16"), (96, "f16"))]
QUERIES = [case([100, 130], [60, 200], dim=dim, heads=(4, 2), dtype=dtype) for dim, dtype in ((32, "f16"), (64, "f16"), (64, "f32"), (128, "bf16"), (128, "f32"), (192, "f16"))]
# The form follows the length that the rows are said to have: up to FEW the queries are divided, from MANY on the keys.
HINTED = [case([40] * 16, [(1990 if s == 5 else 60 + 7 * s) for s in range(16)], dim=dim, heads=(16, 4), dtype=dtype) for dim, dtype in ((64, "bf16"), (128, "f32"))]
FEW, MANY = (0, 1, 256), (1990, 1 << 20, 2 ** 32 - 1)
