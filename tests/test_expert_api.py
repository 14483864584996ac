"""CPU tests of the expert-layer operators' boundary: exported names, phase 1 checks, plans handed to the wrong entry.
No kernel runs (phase 1 is host-only, and a refused phase 2 launches nothing)."""
import ctypes
import os
import re
import subprocess

import pytest

from test_abi import INC, FakeTensor, phase1

HEADER = os.path.join(INC, "aclnnop", "aclnn_block_quant_moe.h")
OK, NULL, BAD = 0, 161001, 161002
i64, cbool = ctypes.c_int64, ctypes.c_bool


def names():
    return re.findall(r"^B200_ACLNN_RUN\((\w+)\)", open(HEADER).read(), re.M)


def test_every_declared_name_is_exported(pkg):
    lib = ctypes.CDLL(pkg.LIB_PATH)
    assert len(names()) == 8
    for n in names():
        assert hasattr(lib, n) and hasattr(lib, n + "GetWorkspaceSize"), n
    out = subprocess.run(["nm", "-g", "--defined-only", os.path.join(os.path.dirname(pkg.LIB_PATH), "libascendcl_qmm.a")],
                         stdout=subprocess.PIPE, text=True, check=True).stdout
    assert all(re.search(r"\b%s$" % n, out, re.M) for n in names())


def test_header_compiles_as_c(tmp_path):
    src = tmp_path / "c.c"
    src.write_text('#include "aclnnop/aclnn_ops.h"\nint main(void) { return aclnnB200MoeTokenPermute == 0; }\n')
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-Wno-address", "-I", INC, "-c", str(src), "-o", str(tmp_path / "c.o")], check=True)


def spread(good, variants):
    """The argument list `good` with one argument replaced at a time."""
    for where, value, want in variants:
        args = list(good)
        args[where] = value
        yield args, want


def check(pkg, name, good, variants):
    assert phase1(pkg, name, *good)[0] == OK
    for n, (args, want) in enumerate(spread(good, variants)):
        assert phase1(pkg, name, *args)[0] == want, (name, n)


def test_block_quant_phase1(pkg):
    T = lambda d, t: FakeTensor(pkg, d, t)
    F, H, B, E4, E5, I8 = pkg.ACL_FLOAT, pkg.ACL_FLOAT16, pkg.ACL_BF16, pkg.ACL_FLOAT8_E4M3FN, pkg.ACL_FLOAT8_E5M2, pkg.ACL_INT8
    x, q, s = T([5, 300], B), T([5, 300], E4), T([5, 3], F)
    check(pkg, "aclnnB200BlockQuantFp8", [x, i64(1), q, s], [
        (0, T([5, 300], F), OK), (0, T([5, 300], H), OK), (2, T([5, 300], E5), OK), (3, T([15], F), OK),
        (0, None, NULL), (2, None, NULL), (3, None, NULL),
        (0, T([5, 300], I8), BAD), (2, T([5, 300], I8), BAD), (3, T([5, 3], H), BAD), (1, i64(64), BAD), (1, i64(0), BAD), (1, i64(-1), BAD),
        (2, T([5, 299], E4), BAD), (2, T([4, 300], E4), BAD), (3, T([5, 2], F), BAD), (3, T([1, 3], F), BAD), (0, T([1500], B), BAD)])
    check(pkg, "aclnnB200BlockQuantFp8", [x, i64(128), q, T([1, 3], F)], [(3, s, BAD)])
    assert phase1(pkg, "aclnnB200BlockQuantFp8", T([0, 300], B), i64(1), T([0, 300], E4), T([0, 3], F))[0] == OK
    assert phase1(pkg, "aclnnB200BlockQuantFp8", T([5, 0], B), i64(1), T([5, 0], E4), T([5, 0], F))[0] == OK
    check(pkg, "aclnnB200SwiGluBlockQuantFp8", [T([2, 5, 600], B), T([2, 5, 300], E4), T([2, 5, 3], F)], [
        (0, None, NULL), (0, T([2, 5, 300], B), BAD), (0, T([2, 5, 599], B), BAD), (1, T([5, 2, 300], E4), BAD), (2, T([2, 5, 5], F), BAD)])


def test_block_matmul_phase1(pkg):
    T = lambda d, t: FakeTensor(pkg, d, t)
    F, H, B, E4, E5, L = pkg.ACL_FLOAT, pkg.ACL_FLOAT16, pkg.ACL_BF16, pkg.ACL_FLOAT8_E4M3FN, pkg.ACL_FLOAT8_E5M2, pkg.ACL_INT64
    M, K, N = 7, 200, 300
    x, xs, w, ws, out = T([M, K], E4), T([M, 2], F), T([K, N], E4), T([2, 3], F), T([M, N], B)
    check(pkg, "aclnnB200BlockQuantMatmul", [x, xs, w, ws, cbool(False), out], [
        (0, T([M, K], E5), OK), (2, T([K, N], E5), OK), (5, T([M, N], H), OK), (5, T([M, N], F), OK),
        (0, None, NULL), (1, None, NULL), (2, None, NULL), (3, None, NULL), (5, None, NULL),
        (0, T([M, K], B), BAD), (0, T([M, K + 1], E4), BAD), (1, T([M, 1], F), BAD), (1, T([M, 2], B), BAD), (2, T([N, K], E4), BAD),
        (3, T([3, 2], F), BAD), (3, T([2, 3], B), BAD), (4, cbool(True), BAD), (5, T([M, N + 1], B), BAD), (5, T([M, N], E4), BAD)])
    check(pkg, "aclnnB200BlockQuantMatmul", [x, xs, T([N, K], E4), T([3, 2], F), cbool(True), out], [(3, ws, BAD)])
    assert phase1(pkg, "aclnnB200BlockQuantMatmul", T([0, K], E4), T([0, 2], F), w, ws, cbool(False), T([0, N], B))[0] == OK
    E = 5
    gx = [x, xs, T([E, K, N], E4), T([E, 2, 3], F), T([E], L), cbool(False), out]
    check(pkg, "aclnnB200BlockQuantGroupedMatmul", gx, [
        (4, None, NULL), (4, T([E], pkg.ACL_INT32), BAD), (4, T([E + 1], L), BAD), (2, w, BAD), (3, T([E, 3, 2], F), BAD), (3, T([4, 2, 3], F), BAD),
        (5, cbool(True), BAD)])
    big = 1025
    assert phase1(pkg, "aclnnB200BlockQuantGroupedMatmul", x, xs, T([big, K, N], E4), T([big, 2, 3], F), T([big], L), cbool(False), out)[0] == BAD


def test_permute_phase1(pkg):
    T = lambda d, t: FakeTensor(pkg, d, t)
    F, H, B, E4, L, I = pkg.ACL_FLOAT, pkg.ACL_FLOAT16, pkg.ACL_BF16, pkg.ACL_FLOAT8_E4M3FN, pkg.ACL_INT64, pkg.ACL_INT32
    t, ids, rows, place, counts = T([6, 40], B), T([6, 2], I), T([12, 40], B), T([6, 2], I), T([9], L)
    check(pkg, "aclnnB200MoeTokenPermute", [t, ids, None, rows, None, place, counts], [
        (1, T([6, 2], L), OK), (3, T([20, 40], B), OK), (2, T([6, 3], F), NULL), (4, T([12, 3], F), NULL),
        (0, None, NULL), (1, None, NULL), (3, None, NULL), (5, None, NULL), (6, None, NULL),
        (0, T([6, 40], I), BAD), (0, T([5, 40], B), BAD), (1, T([6, 2], F), BAD), (3, T([11, 40], B), BAD), (3, T([12, 40], H), BAD), (3, T([12, 41], B), BAD),
        (5, T([6, 2], L), BAD), (5, T([6, 3], I), BAD), (6, T([9], I), BAD), (6, T([1025], L), BAD), (6, T([0], L), BAD)])
    check(pkg, "aclnnB200MoeTokenPermute", [T([6, 40], E4), ids, T([6, 3], F), T([12, 40], E4), T([12, 3], F), place, counts], [
        (2, T([6, 4], F), BAD), (2, T([5, 3], F), BAD), (4, T([11, 3], F), BAD), (2, T([6, 3], H), BAD)])
    assert phase1(pkg, "aclnnB200MoeTokenPermute", T([6, 40], B), T([6, 65], I), None, T([400, 40], B), None, T([6, 65], I), counts)[0] == BAD
    check(pkg, "aclnnB200MoeTokenPermuteGrad", [rows, place, t], [
        (0, None, NULL), (1, None, NULL), (2, None, NULL), (0, T([12, 40], E4), BAD), (2, T([6, 40], H), BAD), (2, T([7, 40], B), BAD), (1, T([6, 2], L), BAD)])


def test_unpermute_phase1(pkg):
    T = lambda d, t: FakeTensor(pkg, d, t)
    F, H, B, L, I = pkg.ACL_FLOAT, pkg.ACL_FLOAT16, pkg.ACL_BF16, pkg.ACL_INT64, pkg.ACL_INT32
    rows, place, probs, out = T([12, 40], B), T([6, 2], I), T([6, 2], F), T([6, 40], B)
    check(pkg, "aclnnB200MoeTokenUnpermute", [rows, place, probs, out], [
        (2, None, OK), (2, T([6, 2], B), OK), (0, T([3, 40], B), OK), (0, None, NULL), (1, None, NULL), (3, None, NULL),
        (1, T([6, 2], L), BAD), (2, T([6, 3], F), BAD), (2, T([6, 2], I), BAD), (3, T([6, 41], B), BAD), (3, T([6, 40], F), BAD)])
    check(pkg, "aclnnB200MoeTokenUnpermuteGrad", [out, rows, place, probs, T([12, 40], B), T([6, 2], F)], [
        (0, None, NULL), (3, None, NULL), (4, None, NULL), (5, None, NULL), (0, T([6, 40], H), BAD), (4, T([11, 40], B), BAD), (5, T([6, 2], B), BAD),
        (3, T([2, 6], F), BAD), (2, T([5, 2], I), BAD)])


def strided(pkg, dims, strides, dtype, addr=0x7F0000000000):
    t = FakeTensor(pkg, dims, dtype, addr)
    lib = pkg.load()
    lib.aclDestroyTensor(ctypes.c_void_p(t.h))
    d, s = (i64 * len(dims))(*dims), (i64 * len(dims))(*strides)
    t.h = lib.aclCreateTensor(d, len(dims), dtype, s, 0, pkg.ACL_FORMAT_ND, d, len(dims), ctypes.c_void_p(addr))
    return t


def test_strided_and_negative_shapes_are_refused(pkg):
    T = lambda d, t: FakeTensor(pkg, d, t)
    B, F, E4, I = pkg.ACL_BF16, pkg.ACL_FLOAT, pkg.ACL_FLOAT8_E4M3FN, pkg.ACL_INT32
    assert phase1(pkg, "aclnnB200BlockQuantFp8", strided(pkg, [5, 300], [512, 1], B), i64(1), T([5, 300], E4), T([5, 3], F))[0] == BAD
    assert phase1(pkg, "aclnnB200BlockQuantMatmul", T([7, 200], E4), T([7, 2], F), strided(pkg, [200, 300], [1, 200], E4), T([2, 3], F), cbool(False),
                  T([7, 300], B))[0] == BAD
    assert phase1(pkg, "aclnnB200MoeTokenUnpermute", T([12, 40], B), strided(pkg, [6, 2], [1, 6], I), None, T([6, 40], B))[0] == BAD
    assert phase1(pkg, "aclnnB200BlockQuantFp8", T([-5, 300], B), i64(1), T([-5, 300], E4), T([-5, 3], F))[0] == BAD


def plan(pkg, name, *args):
    lib = pkg.load()
    ws, ex = ctypes.c_uint64(0), ctypes.c_void_p(0)
    assert getattr(lib, name + "GetWorkspaceSize")(*[ctypes.c_void_p(a.h) if isinstance(a, FakeTensor) else a for a in args], ctypes.byref(ws), ctypes.byref(ex)) == OK
    return ex


def test_phase2_refuses_before_launching(pkg):
    """A plan of another operator, a missing pointer, and outputs that overlap are refused on the host."""
    lib = pkg.load()
    B, F, E4, I, L = pkg.ACL_BF16, pkg.ACL_FLOAT, pkg.ACL_FLOAT8_E4M3FN, pkg.ACL_INT32, pkg.ACL_INT64
    at = lambda d, t, a: FakeTensor(pkg, d, t, a)
    run = lambda name, ex: getattr(lib, name)(None, ctypes.c_uint64(0), ex, None)
    x, q, s = at([4, 256], B, 0x10000), at([4, 256], E4, 0x20000), at([4, 2], F, 0x30000)
    args = (x, i64(1), q, s)
    assert run("aclnnB200MoeTokenPermute", plan(pkg, "aclnnB200BlockQuantFp8", *args)) == BAD
    assert run("aclnnQuantMatmul", plan(pkg, "aclnnB200BlockQuantFp8", *args)) == BAD
    assert run("aclnnB200BlockQuantFp8", None) == NULL
    assert run("aclnnB200BlockQuantFp8", plan(pkg, "aclnnB200BlockQuantFp8", at([4, 256], B, 0), i64(1), q, s)) == NULL
    assert run("aclnnB200BlockQuantFp8", plan(pkg, "aclnnB200BlockQuantFp8", x, i64(1), at([4, 256], E4, 0x10400), s)) == BAD    # codes over x
    assert run("aclnnB200BlockQuantFp8", plan(pkg, "aclnnB200BlockQuantFp8", x, i64(1), q, at([4, 2], F, 0x20010))) == BAD       # scales over codes
    rows, place, probs, out = at([8, 64], B, 0x10000), at([4, 2], I, 0x20000), at([4, 2], F, 0x30000), at([4, 64], B, 0x10100)
    assert run("aclnnB200MoeTokenUnpermute", plan(pkg, "aclnnB200MoeTokenUnpermute", rows, place, probs, out)) == BAD
    assert run("aclnnB200MoeTokenUnpermute", plan(pkg, "aclnnB200MoeTokenUnpermute", rows, place, at([4, 2], F, 0), at([4, 64], B, 0x40000))) == NULL
    assert run("aclnnB200BlockQuantFp8", plan(pkg, "aclnnB200BlockQuantFp8", x, i64(1), q, at([4, 2], F, 0x30002))) == BAD       # off a float's boundary
    # an empty batch needs no pointers and launches nothing
    assert run("aclnnB200MoeTokenUnpermute", plan(pkg, "aclnnB200MoeTokenUnpermute", at([0, 64], B, 0), at([0, 2], I, 0), None, at([0, 64], B, 0))) == OK
    assert run("aclnnB200BlockQuantMatmul", plan(pkg, "aclnnB200BlockQuantMatmul", at([0, 64], E4, 0), at([0, 1], F, 0), at([64, 32], E4, 0x1000),
                                                 at([1, 1], F, 0x2000), cbool(False), at([0, 32], B, 0))) == OK


def test_both_phases_in_one_call(pkg):
    lib = pkg.load()
    B, F, E4 = pkg.ACL_BF16, pkg.ACL_FLOAT, pkg.ACL_FLOAT8_E4M3FN
    vp, u64 = ctypes.c_void_p, ctypes.c_uint64

    def run(op, tensors, addrs, option=0, count=None):
        hs = (vp * max(1, len(tensors)))(*[t.h if t else None for t in tensors])
        return lib.aclnnB200RunExpertOp(ctypes.c_int(op), hs, (vp * max(1, len(addrs)))(*addrs), u64(len(tensors) if count is None else count),
                                        i64(option), vp(0))

    x, q, s = FakeTensor(pkg, [4, 256], B), FakeTensor(pkg, [4, 256], E4), FakeTensor(pkg, [4, 2], F)
    got = vp(0)
    assert run(0, [x, q, s], [0x10000, 0x10400, 0x30000], 1) == BAD             # codes over x
    for t, want in ((x, 0x10000), (q, 0x10400), (s, 0x30000)):
        assert lib.aclGetRawTensorAddr(vp(t.h), ctypes.byref(got)) == OK and got.value == want
    assert run(0, [x, q, s], [0, 0x20000, 0x30000], 1) == NULL
    assert run(0, [x, q, s], [0x10000, 0x20000, 0x30000], 64) == BAD            # phase 1's refusal
    assert run(0, [x, None, s], [0x10000, 0x20000, 0x30000], 1) == NULL
    assert run(0, [x, q, s], [0x10000, 0x20000, 0x30000], 1, count=2) == BAD
    for op in (-1, 8, 1 << 20):
        assert run(op, [x, q, s], [0x10000, 0x20000, 0x30000]) == BAD
    assert lib.aclnnB200RunExpertOp(ctypes.c_int(0), None, None, u64(3), i64(1), vp(0)) == NULL
    rows, place, out = FakeTensor(pkg, [0, 64], B), FakeTensor(pkg, [0, 2], pkg.ACL_INT32), FakeTensor(pkg, [0, 64], B)
    assert run(5, [rows, place, out], [0, 0, 0]) == OK and run(6, [rows, place, None, out], [0, 0, 0, 0]) == OK     # empty: nothing is launched
    w = [FakeTensor(pkg, d, t) for d, t in (([0, 64], E4), ([0, 1], F), ([64, 32], E4), ([1, 1], F), ([0, 32], B))]
    assert run(2, w, [0, 0, 0x1000, 0x2000, 0]) == OK and run(2, w, [0, 0, 0x1000, 0x2000, 0], 1) == BAD            # [K, N], not [N, K]


def test_wrappers_refuse_what_the_abi_would_misread(pkg):
    import torch
    with pytest.raises(ValueError):
        pkg.block_quant_fp8(torch.zeros(4, 128))
    with pytest.raises(ValueError):
        pkg.moe_token_permute(torch.zeros(4, 128), torch.zeros(4, 2, dtype=torch.int32), 4)
