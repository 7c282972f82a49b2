"""dot_general of 8-bit integers with 32-bit sums through the compiler: plan and refusals on the CPU, results on
the GPU equal to the oracle's (integers, so exactly), alone and with the scales of a quantised linear layer
around it."""
import numpy as np
import pytest

from conftest import RTOL_F32, assert_close
from oracle.interp import run as oracle_run
from pjrt_b200.shlo import Builder
from test_compiler import report

CASES = {  # name: lhs shape, rhs shape, batch dims, contracting dims
    "k_major": ((48, 256), (130, 256), ((), ()), ([1], [1])),
    "one_token": ((1, 768), (2304, 768), ((), ()), ([1], [1])),
    "mn_major": ((300, 64), (64, 200), ((), ()), ([1], [0])),
    "odd": ((37, 75), (75, 53), ((), ()), ([1], [0])),
    "batched": ((3, 70, 96), (3, 40, 96), ([0], [0]), ([2], [2])),
    "batched_mn": ((2, 33, 40), (2, 40, 50), ([0], [0]), ([2], [1])),
    "two_dims": ((20, 4, 32), (30, 4, 32), ((), ()), ([1, 2], [1, 2])),
    "wide": ((600, 1024), (1024, 520), ((), ()), ([1], [0])),
}


def program(name, out="i32"):
    ls, rs, batch, contract = CASES[name]
    b = Builder("jit_dot_i8")
    x, w = b.arg(ls, "i8"), b.arg(rs, "i8")
    return b.text([b.dot_general(x, w, batch=batch, contract=contract, out_dtype=out)])


def inputs(name, seed=0):
    rng = np.random.default_rng(seed)
    return [rng.integers(-128, 128, s, dtype=np.int8) for s in CASES[name][:2]]


def test_oracle_sums_wide():
    x, w = inputs("odd")
    (r,) = oracle_run(program("odd"), [x, w])
    assert r.dtype == np.int32
    np.testing.assert_array_equal(r, x.astype(np.int64) @ w.astype(np.int64))


@pytest.mark.parametrize("name,copies", [("k_major", 0), ("one_token", 0), ("mn_major", 1), ("odd", 2), ("batched", 0), ("batched_mn", 2),
                                         ("two_dims", 0), ("wide", 1)])
def test_plan(lib_path, name, copies):
    rc, rep = report(lib_path, program(name))
    steps = [l for l in rep.splitlines() if l.startswith("  [")]
    assert rc == 0, rep
    assert sum(" i8" in l and "gemm" in l for l in steps) == 1 and sum("transpose" in l for l in steps) == copies, rep


@pytest.mark.parametrize("out", ["i8", "f32"])
def test_other_results_are_refused(lib_path, out):
    rc, rep = report(lib_path, program("k_major", out))
    assert rc != 0 and "dot_general on non-float operands" in rep, rep


def test_deep_sums_are_refused(lib_path):
    b = Builder("jit_deep")
    x, w = b.arg((1, 131072), "i8"), b.arg((1, 131072), "i8")
    rc, rep = report(lib_path, b.text([b.dot_general(x, w, contract=([1], [1]), out_dtype="i32")]))
    assert rc != 0 and "at most 131071" in rep, rep


@pytest.mark.gpu
@pytest.mark.parametrize("name", sorted(CASES))
def test_sums_equal_the_oracle(client, name):
    ins = inputs(name, 3)
    (ref,) = oracle_run(program(name), ins)
    (got,) = client.run(program(name), ins)
    np.testing.assert_array_equal(got, ref)


def scaled_program(m, n, k):
    """f32(x . w^T) * row scale * column scale: the product's sums and a generated kernel behind it."""
    b = Builder("jit_linear_i8")
    x, w, sx, sw = b.arg((m, k), "i8"), b.arg((n, k), "i8"), b.arg((m,), "f32"), b.arg((n,), "f32")
    y = b.convert(b.dot_general(x, w, contract=([1], [1]), out_dtype="i32"), "f32")
    return b.text([y * b.broadcast_in_dim(sx, (m, n), [0]) * b.broadcast_in_dim(sw, (m, n), [1])])


def test_scaled_plan(lib_path):
    rc, rep = report(lib_path, scaled_program(90, 140, 320))
    steps = [l for l in rep.splitlines() if l.startswith("  [")]
    assert rc == 0 and len(steps) == 2, rep


@pytest.mark.gpu
def test_scaled_linear_layer(client):
    m, n, k = 90, 140, 320
    text = scaled_program(m, n, k)
    rng = np.random.default_rng(5)
    ins = [rng.integers(-128, 128, (m, k), dtype=np.int8), rng.integers(-128, 128, (n, k), dtype=np.int8),
           rng.random(m).astype(np.float32), rng.random(n).astype(np.float32)]
    assert_close(client.run(text, ins)[0], oracle_run(text, ins)[0], RTOL_F32)


def computed_program(m, n, k):
    """Operands that the program computes: x rounded to 8 bits, w transposed."""
    b = Builder("jit_computed_i8")
    x, w = b.arg((m, k), "f32"), b.arg((k, n), "i8")
    q = b.convert(x * 2.0, "i8")
    return b.text([b.dot_general(q, b.transpose(w, [1, 0]), contract=([1], [1]), out_dtype="i32"), q])


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(37, 53, 75), (1, 40, 33), (130, 64, 64)])
def test_computed_operands(client, m, n, k):
    rng = np.random.default_rng(6)
    ins = [rng.integers(-60, 61, (m, k)).astype(np.float32), rng.integers(-128, 128, (k, n), dtype=np.int8)]
    text = computed_program(m, n, k)
    for got, ref in zip(client.run(text, ins), oracle_run(text, ins)):
        np.testing.assert_array_equal(got, ref)


@pytest.mark.parametrize("m,n", [(2147483392, 1), (1, 2147483392)])
def test_more_rows_than_a_launch_takes_are_refused(lib_path, m, n):
    b = Builder("jit_tall")
    x, w = b.arg((m, 16), "i8"), b.arg((n, 16), "i8")
    rc, rep = report(lib_path, b.text([b.dot_general(x, w, contract=([1], [1]), out_dtype="i32")]))
    assert rc != 0 and "at most 2147483391 rows" in rep, rep


def test_most_rows(lib_path):
    b = Builder("jit_tall")
    x, w = b.arg((2147483391, 16), "i8"), b.arg((1, 16), "i8")
    rc, rep = report(lib_path, b.text([b.dot_general(x, w, contract=([1], [1]), out_dtype="i32")]))
    assert rc == 0, rep
