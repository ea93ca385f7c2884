"""The tests of attention over pages run every form of its kernel that a call can take."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

import paged_plan


def test_every_form_is_reached():
    reached = {paged_plan.form_of(form, D, paged_plan.B, paged_plan.H, group, T, page, -(-table // page))
               for form in paged_plan.ROW for D in (64, 128) for group, T in paged_plan.ROWS for page in paged_plan.PAGES for table in paged_plan.TABLES}
    assert reached == paged_plan.all_forms(), paged_plan.all_forms() - reached


@pytest.mark.parametrize("form", list(paged_plan.ROW))
@pytest.mark.parametrize("D", [64, 128])
def test_the_rules_are_the_librarys(akv_lib, form, D):
    """The workspace says how many tiles a unit has, and whether clusters take it (none then)."""
    from alignedkv_b200 import _lib
    sms = torch.cuda.get_device_properties(0).multi_processor_count if torch.cuda.is_available() else 148
    code = {"fp16": 0, "e4m3": 1, "e2m1": 2}[form]
    for B, H in ((1, 1), (4, 8), (13, 4), (20, 8), (300, 2)):
        for rows in (1, 8, 9, 20, 32, 64):
            for page in (16, 256):
                for table in (256, 512, 6144, 6208, 200000):
                    width = -(-table // page)
                    pool = _lib.Pool(None, None, None, None, None, None, code, 1, page, H, D)
                    want = paged_plan.plan(form, D, B, H, rows, 1, page, width, sms)[2]
                    assert akv_lib.akv_paged_scratch_bytes(ctypes.byref(pool), B, width, rows, 1) == want, (B, H, rows, page, table)
