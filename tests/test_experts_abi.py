"""CPU checks of the experts' operators: the status codes of the C entry points and the Python module's refusals.

No call here reaches a kernel launch: each fails its checks, sizes a buffer, or has nothing to do.
"""
import ctypes
import re
import shutil
import subprocess

import pytest
import torch

import ops_sparse
from ops_sparse import _lib, experts
from ops_sparse._lib import DataType, Operation, Status

F32, F16, BF16, I8 = (int(DataType.FLOAT), int(DataType.FLOAT16), int(DataType.BF16), int(DataType.INT8))
NT, NN = int(Operation.TRANSPOSE), int(Operation.NON_TRANSPOSE)
P = 4096  # stands for a device pointer: never followed


@pytest.fixture(scope="module")
def lib():
    return _lib.lib()


@pytest.fixture(scope="module")
def handle(lib):
    h = ctypes.c_void_p(0)
    assert lib.aclsparseCreate(ctypes.byref(h)) == Status.SUCCESS
    yield h
    lib.aclsparseDestroy(h)


def route(**kw):
    a = dict(tokens=4, experts=8, k=2, logits=P, ld=8, type=F32, normalize=1, weights=P, ids=P, offsets=P, rows=P,
             places=P, buffer=P)
    a.update(kw)
    return list(a.values())


def route_grad(**kw):
    a = dict(tokens=4, experts=8, k=2, logits=P, ld=8, type=F32, normalize=0, weights=P, ids=P, grad=P, out=P, ldg=8)
    a.update(kw)
    return list(a.values())


def plan(**kw):
    a = dict(tokens=4, experts=8, k=2, ids=P, offsets=P, rows=P, places=P, buffer=P)
    a.update(kw)
    return list(a.values())


def grouped(**kw):
    a = dict(op=NT, groups=2, rows=4, n=8, k=16, offsets=P, index=P, rows_a=4, a=P, lda=16, b=P, ldb=16, stride=128,
             type=BF16, c=P, ldc=8, ctype=BF16)
    a.update(kw)
    return list(a.values())


def scaled(**kw):
    a = dict(groups=2, rows=4, n=8, k=16, offsets=P, index=P, rows_a=4, a=P, lda=16, sa=P, b=P, ldb=16, stride=128,
             sb=P, c=P, ldc=8, ctype=BF16)
    a.update(kw)
    return list(a.values())


def grad(**kw):
    a = dict(groups=2, rows=4, n=8, k=16, offsets=P, index=P, rows_x=4, g=P, ldg=8, x=P, ldx=16, type=F16, w=P, ldw=16,
             stride=128, wtype=F16)
    a.update(kw)
    return list(a.values())


def combine(**kw):
    a = dict(tokens=4, k=2, width=8, rows=8, places=P, weights=P, y=P, ldy=8, ytype=F16, out=P, ldo=8, otype=F16)
    a.update(kw)
    return list(a.values())


def combine_grad(**kw):
    a = dict(tokens=4, k=2, width=8, rows=8, groups=2, offsets=P, places=P, weights=P, y=P, ldy=8, go=P, ldo=8,
             type=F16, gy=P, ldgy=8, gw=P)
    a.update(kw)
    return list(a.values())


INVALID, UNSUPPORTED, OK = Status.INVALID_VALUE, Status.NOT_SUPPORTED, Status.SUCCESS
CASES = [
    ("aclsparseRoute", route, [
        (dict(tokens=-1), INVALID), (dict(experts=0), INVALID), (dict(k=0), INVALID), (dict(k=9), INVALID),
        (dict(experts=1025, ld=1025), UNSUPPORTED), (dict(experts=100, k=65, ld=100), UNSUPPORTED),
        (dict(tokens=2**31), UNSUPPORTED), (dict(type=I8), UNSUPPORTED), (dict(logits=0), INVALID),
        (dict(weights=0), INVALID), (dict(ids=0), INVALID), (dict(offsets=0), INVALID), (dict(rows=0), INVALID),
        (dict(places=0), INVALID), (dict(buffer=0), INVALID), (dict(ld=7), INVALID)]),
    ("aclsparseExpertPlan", plan, [
        (dict(tokens=-1), INVALID), (dict(k=9), INVALID), (dict(ids=0), INVALID), (dict(offsets=0), INVALID),
        (dict(buffer=0), INVALID), (dict(experts=2000), UNSUPPORTED)]),
    ("aclsparseRouteGrad", route_grad, [
        (dict(k=9), INVALID), (dict(type=I8), UNSUPPORTED), (dict(logits=0), INVALID), (dict(grad=0), INVALID),
        (dict(out=0), INVALID), (dict(ldg=7), INVALID), (dict(ld=7), INVALID), (dict(tokens=0), OK)]),
    ("aclsparseGroupedMM", grouped, [
        (dict(op=2), UNSUPPORTED), (dict(groups=0), INVALID), (dict(rows=-1), INVALID), (dict(n=-1), INVALID),
        (dict(k=-1), INVALID), (dict(rows=2**31 - 64, rows_a=2**31 - 64), UNSUPPORTED), (dict(offsets=0), INVALID),
        (dict(n=2**31 - 64, ldc=2**31), UNSUPPORTED), (dict(k=2**31 - 64, lda=2**31, ldb=2**31), UNSUPPORTED),
        (dict(index=0, rows_a=3), INVALID), (dict(rows_a=0), INVALID), (dict(type=F32), UNSUPPORTED),
        (dict(type=I8), UNSUPPORTED), (dict(ctype=F16), UNSUPPORTED), (dict(lda=15), INVALID), (dict(ldb=15), INVALID),
        (dict(op=NN, ldb=7), INVALID), (dict(ldc=7), INVALID), (dict(stride=-1), INVALID), (dict(c=0), INVALID),
        (dict(a=0), INVALID), (dict(b=0), INVALID), (dict(rows=0), OK), (dict(n=0), OK)]),
    ("aclsparseGroupedMMScaled", scaled, [
        (dict(groups=0), INVALID), (dict(k=131072, lda=131072, ldb=131072), UNSUPPORTED), (dict(ctype=I8), UNSUPPORTED),
        (dict(sa=0), INVALID), (dict(sb=0), INVALID), (dict(lda=15), INVALID), (dict(ldc=7), INVALID),
        (dict(rows=0), OK)]),
    ("aclsparseGroupedMMGrad", grad, [
        (dict(type=F32, wtype=F32), UNSUPPORTED), (dict(wtype=BF16), UNSUPPORTED), (dict(ldg=7), INVALID),
        (dict(ldx=15), INVALID), (dict(ldw=15), INVALID), (dict(stride=127), INVALID),
        (dict(stride=16, ldw=31), INVALID), (dict(w=0), INVALID), (dict(g=0), INVALID), (dict(x=0), INVALID),
        (dict(n=0), OK), (dict(k=0), OK)]),
    ("aclsparseCombine", combine, [
        (dict(k=0), INVALID), (dict(k=65), UNSUPPORTED), (dict(ytype=BF16), UNSUPPORTED),
        (dict(otype=F32, ytype=F32), UNSUPPORTED), (dict(ldy=7), INVALID), (dict(ldo=7), INVALID),
        (dict(places=0), INVALID), (dict(out=0), INVALID), (dict(y=0), INVALID), (dict(tokens=0), OK),
        (dict(width=0), OK)]),
    ("aclsparseCombineGrad", combine_grad, [
        (dict(groups=0), INVALID), (dict(type=F32), UNSUPPORTED), (dict(ldo=7), INVALID), (dict(ldgy=7), INVALID),
        (dict(ldy=7), INVALID), (dict(offsets=0), INVALID), (dict(places=0), INVALID), (dict(y=0), INVALID),
        (dict(go=0), INVALID), (dict(gy=0, gw=0), OK), (dict(tokens=0, rows=0), OK)]),
]


@pytest.mark.parametrize("name,args,changes", CASES, ids=[c[0] for c in CASES])
def test_status_codes(lib, handle, name, args, changes):
    fn = getattr(lib, name)
    assert fn(None, *args()) == Status.HANDLE_IS_NULLPTR
    for change, status in changes:
        assert fn(handle, *args(**change)) == status, (name, change)


@pytest.mark.parametrize("name,args", [("aclsparseGroupedMM", grouped), ("aclsparseGroupedMMScaled", scaled),
                                       ("aclsparseGroupedMMGrad", grad)])
def test_more_groups_than_a_scan_can_count_are_refused(lib, handle, name, args):
    # the kernels' scans go over the groups 64 at a time in int32, and their last step has to fit it
    for groups in (2**31 - 4096, 2**31 - 64, 2**31 - 1, 2**40):
        assert getattr(lib, name)(handle, *args(groups=groups, stride=0 if name != "aclsparseGroupedMMGrad" else 128)) \
            == UNSUPPORTED, groups


def test_grids_of_too_many_threads_are_refused(lib, handle):
    # a grid's dimension takes fewer than 2^32 threads: these need more workgroups than that, though fewer than 2^31
    for name, args in (
            ("aclsparseGroupedMM", grouped(groups=2**18, rows=2**18, rows_a=2**18, n=2**14, ldc=2**14)),
            ("aclsparseGroupedMM", grouped(op=NN, groups=2**18, rows=2**18, rows_a=2**18, n=2**14, ldb=2**14, ldc=2**14)),
            ("aclsparseGroupedMM", grouped(groups=2, rows=2**25, rows_a=2**25, n=2**14, ldc=2**14)),
            ("aclsparseGroupedMMScaled", scaled(groups=2**18, rows=2**18, rows_a=2**18, n=2**14, ldc=2**14)),
            ("aclsparseGroupedMMGrad", grad(groups=2**10, n=2**17, k=2**13, ldg=2**17, ldx=2**13, ldw=2**13,
                                            stride=2**30))):
        assert getattr(lib, name)(handle, *args) == UNSUPPORTED, (name, args)


def combine_grad_any(**kw):
    a = dict(tokens=4, k=2, width=8, rows=8, places=P, weights=P, y=P, ldy=8, go=P, ldo=8, type=F16, gy=P, ldgy=8, gw=P,
             buffer=P, listed=0)
    a.update(kw)
    return list(a.values())


def test_status_codes_of_the_combination_that_lists(lib, handle):
    # as the one that does not, and the buffer
    for change, status in dict((name, changes) for name, _, changes in CASES)["aclsparseCombine"]:
        assert lib.aclsparseCombineAndList(handle, *combine(**change), P) == status, change
    assert lib.aclsparseCombineAndList(handle, *combine(), None) == INVALID
    assert lib.aclsparseCombineAndList(handle, *combine(tokens=0), None) == OK
    assert lib.aclsparseCombineAndList(None, *combine(), P) == Status.HANDLE_IS_NULLPTR


def test_status_codes_of_the_gradient_for_any_places(lib, handle):
    fn = lib.aclsparseCombineGradAny
    assert fn(None, *combine_grad_any()) == Status.HANDLE_IS_NULLPTR
    for change, status in [
            (dict(tokens=-1), INVALID), (dict(k=0), INVALID), (dict(k=65), UNSUPPORTED), (dict(rows=-1), INVALID),
            (dict(rows=2**31), UNSUPPORTED), (dict(tokens=2**30), UNSUPPORTED), (dict(type=F32), UNSUPPORTED),
            (dict(ldo=7), INVALID), (dict(ldgy=7), INVALID), (dict(ldy=7), INVALID), (dict(places=0), INVALID),
            (dict(y=0), INVALID), (dict(go=0), INVALID), (dict(buffer=0), INVALID), (dict(gy=0, gw=0, buffer=0), OK),
            (dict(tokens=0, rows=0), OK)]:
        assert fn(handle, *combine_grad_any(**change)) == status, change


def test_buffer_size_of_the_gradient_for_any_places(lib, handle):
    size = ctypes.c_size_t(0)
    fn = lib.aclsparseCombineGradAny_bufferSize
    for tokens, k, rows in ((0, 1, 0), (1, 1, 1), (100, 3, 7), (16384, 8, 2**31 - 1), (2**25, 63, 5)):
        assert fn(handle, tokens, k, rows, ctypes.byref(size)) == OK
        assert 4 * (rows + tokens * k) <= size.value <= 4 * (rows + tokens * k) + 192 and size.value % 64 == 0
    assert fn(handle, 4, 2, 8, None) == INVALID
    assert fn(handle, 4, 65, 8, ctypes.byref(size)) == UNSUPPORTED
    assert fn(None, 4, 2, 8, ctypes.byref(size)) == Status.HANDLE_IS_NULLPTR


def test_buffer_size(lib, handle):
    size = ctypes.c_size_t(0)
    for tokens, experts, k in ((0, 1, 1), (1, 8, 2), (64, 64, 8), (16384, 128, 8), (10**6, 1024, 2)):
        assert lib.aclsparseRoute_bufferSize(handle, tokens, experts, k, ctypes.byref(size)) == OK
        # one count per expert and workgroup, of which there are 256 at most
        assert size.value > 0 and size.value % 64 == 0 and size.value <= 256 * experts * 4 + 64
    assert lib.aclsparseRoute_bufferSize(handle, 4, 8, 2, None) == INVALID
    assert lib.aclsparseRoute_bufferSize(handle, 4, 8, 9, ctypes.byref(size)) == INVALID


def test_module_matches_the_sources():
    from ops_sparse.build import source_hash

    assert experts._module().build_id == source_hash()


def test_cpu_tensors_are_refused():
    i = torch.zeros(4, 2, dtype=torch.int32)
    p = ops_sparse.ExpertPlan(torch.zeros(3, dtype=torch.int32), torch.zeros(8, dtype=torch.int32), i)
    h, w = torch.zeros(8, 16, dtype=torch.float16), torch.zeros(2, 8, 16, dtype=torch.float16)
    for call in (lambda: ops_sparse.route(torch.zeros(4, 8), 2), lambda: ops_sparse.expert_plan(i, 4),
                 lambda: ops_sparse.grouped_mm(h, w, p), lambda: ops_sparse.combine(h, p),
                 lambda: ops_sparse.grouped_mm_scaled(h.to(torch.int8), torch.ones(8), w[0].to(torch.int8),
                                                      torch.ones(8))):
        with pytest.raises(ValueError, match="ROCm device"):
            call()


def test_forward_mode_is_refused():
    # before the device is looked at, so tensors of the host show it
    i = torch.zeros(4, 2, dtype=torch.int32)
    p = ops_sparse.ExpertPlan(torch.zeros(3, dtype=torch.int32), torch.zeros(8, dtype=torch.int32), i)
    h, w = torch.zeros(8, 16, dtype=torch.float16), torch.zeros(2, 8, 16, dtype=torch.float16)
    one, logits = torch.ones(8), torch.zeros(4, 8)
    with torch.autograd.forward_ad.dual_level():
        def dual(t):
            return torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))

        for call in (lambda: ops_sparse.route(dual(logits), 2), lambda: ops_sparse.grouped_mm(dual(h), w, p),
                     lambda: ops_sparse.grouped_mm(h, dual(w), p), lambda: ops_sparse.combine(dual(h), p),
                     lambda: ops_sparse.combine(h, p, dual(torch.ones(4, 2))),
                     lambda: ops_sparse.grouped_mm_scaled(h.to(torch.int8), dual(one), w[0].to(torch.int8), one),
                     lambda: ops_sparse.grouped_mm_scaled(h.to(torch.int8), one, w[0].to(torch.int8), dual(one))):
            with pytest.raises(NotImplementedError, match="forward"):
                call()


def other_uses_of_m0(lines):
    """Lines that name m0, but those that set it for the copy to LDS right behind them."""
    found = []
    for i, line in enumerate(lines):
        if re.search(r"\bm0\b", line):
            copy = (re.fullmatch(r"s_mov_b32 m0, s\d+", line) and lines[i + 1] == "s_nop 0"
                    and lines[i + 2].startswith("global_load_lds_dwordx4 "))
            if not copy:
                found.append(line)
    return found


def test_the_copies_to_lds_are_the_only_use_of_m0(tmp_path):
    # The grouped products set m0 in assembly that cannot say so: it is a reserved register, whose clobber the compiler
    # does not heed.  That holds as long as the compiler itself needs m0 nowhere in their code.
    tool = "/opt/rocm/llvm/bin/llvm-objdump"
    shutil.copy(_lib.LIB_PATH, tmp_path / "lib.so")
    subprocess.run([tool, "--offloading", "lib.so"], cwd=tmp_path, check=True, capture_output=True)
    images = [f for f in tmp_path.iterdir() if f.name.endswith("gfx950") and b"GroupedTileKernel" in f.read_bytes()]
    assert len(images) == 1
    text = subprocess.run([tool, "-d", "--no-show-raw-insn", images[0].name], cwd=tmp_path, check=True,
                          capture_output=True, text=True).stdout
    lines = [line.split("//")[0].strip() for line in text.splitlines()]
    assert sum(line.startswith("global_load_lds_dwordx4 ") for line in lines) > 100
    assert other_uses_of_m0(lines) == []
    assert other_uses_of_m0(lines + ["s_mov_b32 m0, -1", "ds_read_b32 v0, v1", ""]) == ["s_mov_b32 m0, -1"]
