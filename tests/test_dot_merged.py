"""dot_general that contracts several dimensions, or none, where K is no multiple of what a row's pitch has to be a
multiple of: the copies lie in rows of all contracted dimensions together.  Where the copies' rows begin is read
off the generated source on the CPU; results on the GPU against the oracle."""
import re

import numpy as np
import pytest

from conftest import RTOL_BF16, assert_close
from oracle.interp import run as oracle_run
from pjrt_b200.shlo import Builder
from test_compiler import report

CASES = {  # name: lhs shape, rhs shape, batch dims, contracting dims, K
    "two_dims": ((20, 3, 5), (30, 3, 5), ((), ()), ([1, 2], [1, 2]), 15),
    "two_dims_swapped": ((20, 5, 3), (30, 3, 5), ((), ()), ([2, 1], [1, 2]), 15),
    "two_dims_first": ((3, 7, 21), (3, 7, 33), ((), ()), ([0, 1], [0, 1]), 21),
    "two_dims_batched": ((4, 19, 3, 3), (4, 3, 3, 17), ([0], [0]), ([2, 3], [1, 2]), 9),
    "three_dims": ((9, 3, 5, 11), (13, 3, 5, 11), ((), ()), ([1, 2, 3], [1, 2, 3]), 165),
    "outer": ((21,), (33,), ((), ()), ([], []), 1),
    "outer_two": ((5, 7), (3, 11), ((), ()), ([], []), 1),
    "outer_batched": ((4, 13), (4, 19), ([0], [0]), ([], []), 1),
}


def program(name, dtype, out):
    ls, rs, batch, contract, _ = CASES[name]
    b = Builder("jit_dot_merged")
    x, w = b.arg(ls, dtype), b.arg(rs, dtype)
    return b.text([b.dot_general(x, w, batch=batch, contract=contract, out_dtype=out)])


def check_pitches(lib_path, tmp_path, monkeypatch, name, dtype, out, unit):
    """Both operands are copied to rows of K elements, the multiple of `unit` that follows apart."""
    dump = tmp_path / "kernels.cu"
    monkeypatch.setenv("B200_DUMP_CUDA", str(dump))
    rc, rep = report(lib_path, program(name, dtype, out))
    assert rc == 0, rep
    k = CASES[name][4]
    rows = re.findall(r"out0\[\(i / (\d+)LL\) \* (\d+)LL \+ i % (\d+)LL\]", dump.read_text())
    assert rows == 2 * [(str(k), str((k + unit - 1) // unit * unit), str(k))], rows


@pytest.mark.parametrize("name", sorted(CASES))
def test_pitches(lib_path, tmp_path, monkeypatch, name):
    check_pitches(lib_path, tmp_path, monkeypatch, name, "bf16", "f32", 8)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("name", sorted(CASES))
def test_products(client, name, dtype):
    import ml_dtypes
    rng = np.random.default_rng(7)
    ins = [rng.standard_normal(s).astype(ml_dtypes.bfloat16 if dtype == "bf16" else np.float16) for s in CASES[name][:2]]
    text = program(name, dtype, "f32")
    assert_close(client.run(text, ins)[0], oracle_run(text, ins)[0], RTOL_BF16)


@pytest.mark.parametrize("name", sorted(CASES))
def test_pitches_i8(lib_path, tmp_path, monkeypatch, name):
    check_pitches(lib_path, tmp_path, monkeypatch, name, "i8", "i32", 16)


@pytest.mark.gpu
@pytest.mark.parametrize("name", sorted(CASES))
def test_sums_i8(client, name):
    rng = np.random.default_rng(8)
    ins = [rng.integers(-128, 128, s, dtype=np.int8) for s in CASES[name][:2]]
    text = program(name, "i8", "i32")
    np.testing.assert_array_equal(client.run(text, ins)[0], oracle_run(text, ins)[0])


def no_depth_program():
    b = Builder("jit_no_depth")
    x, w = b.arg((5, 0, 3), "i8"), b.arg((0, 7, 3), "i8")
    return b.text([b.dot_general(x, w, contract=([1, 2], [0, 2]), out_dtype="i32")])


def scalars_program():
    b = Builder("jit_scalars")
    x, w = b.arg((), "i8"), b.arg((), "i8")
    return b.text([b.dot_general(x, w, contract=([], []), out_dtype="i32")])


@pytest.mark.parametrize("text", [no_depth_program(), scalars_program()], ids=["no_depth", "scalars"])
def test_smallest_plans_i8(lib_path, text):
    rc, rep = report(lib_path, text)
    assert rc == 0 and " i8" in rep, rep


@pytest.mark.gpu
def test_smallest_i8(client):
    (got,) = client.run(no_depth_program(), [np.zeros((5, 0, 3), np.int8), np.zeros((0, 7, 3), np.int8)])
    np.testing.assert_array_equal(got, np.zeros((5, 7), np.int32))
    (got,) = client.run(scalars_program(), [np.int8(-128), np.int8(-7)])
    assert int(got) == 896
