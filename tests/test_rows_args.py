"""Refusals of the row products, without a GPU: the argument checks the entry
points call before any launch (hk_rows_args.h), built for the host."""
import os
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
ARG, GEOM, UNSUP = 1, 2, 5

EXPECT = {
    "ok": 0, "ok_order": 0, "ok_no_rows": 0, "ok_one_row_any_stride": 0, "kind_f32": UNSUP, "kind_rice": UNSUP,
    "type": UNSUP, "type_negative": UNSUP, "null_x": ARG, "misaligned_y": ARG, "misaligned_x": ARG, "x_stride": GEOM,
    "y_stride": GEOM, "stride_overflow": GEOM, "too_many": UNSUP, "few_x": GEOM, "no_x": GEOM, "per_row": ARG,
    "null_offsets": ARG, "null_ws": ARG, "misaligned_ws": ARG, "short_ws": ARG, "overlap": ARG, "touching_is_ok": 0,
    "ws_in_x": ARG, "ws_in_y": ARG,
    "g_ok": 0, "g_ok_empty": 0, "g_no_groups": UNSUP, "g_many_groups": UNSUP, "g_many_ids": UNSUP, "g_one_id_more": UNSUP,
    "g_null_ids": ARG,
    "g_null_pos": ARG, "g_null_offsets": ARG, "g_alias": ARG, "g_alias_offsets": ARG, "g_no_ws": ARG, "g_short_ws": ARG,
    "c_ok": 0, "c_ok_in_place": 0, "c_ok_no_x": 0, "c_cols": GEOM, "c_per_row": GEOM, "c_null_pos": ARG, "c_null_w": ARG,
    "c_stride": GEOM, "c_base_few": GEOM, "c_base_overlap": ARG, "c_x_overlap": ARG,
    "b_ok": 0, "b_kind": UNSUP, "b_slots": UNSUP, "b_rank": UNSUP, "a_ok": 0, "a_ok_empty": 0, "a_slot": ARG,
    "a_rank": GEOM, "a_type": UNSUP, "a_null": ARG, "a_misaligned": ARG,
}


@pytest.fixture(scope="module")
def said(tmp_path_factory):
    exe = tmp_path_factory.mktemp("rows_args") / "harness"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-o", str(exe), os.path.join(HERE, "rows_args_harness.cpp")],
                   check=True, capture_output=True, text=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout
    return {name: int(code) for name, code in (line.split() for line in out.splitlines())}


def test_every_case_is_named(said):
    assert set(said) == set(EXPECT)


@pytest.mark.parametrize("name", sorted(EXPECT))
def test_status(said, name):
    assert said[name] == EXPECT[name]


def test_row_types():
    from hawking_amd import rows
    with pytest.raises(ValueError):
        rows._row_type("f64")
