"""CPU checks of the operators of training and serving: status codes of the C entry points, the module's refusals, and
the random numbers that 8-bit moments are rounded by.

No call here reaches a kernel launch: each fails its checks, sizes a buffer, or has nothing to do.
"""
import ctypes
import shutil
import subprocess

import numpy as np
import pytest
import torch

import ops_sparse
from ops_sparse import _lib
from ops_sparse._lib import AdamWOptions, AdamWTensor, DataType, Status

F32, F16, BF16, I8, I32, I64 = (int(getattr(DataType, n)) for n in ("FLOAT", "FLOAT16", "BF16", "INT8", "INT32", "INT64"))
INVALID, UNSUPPORTED, OK = Status.INVALID_VALUE, Status.NOT_SUPPORTED, Status.SUCCESS
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


def quantize(**kw):
    a = dict(rows=4, k=40, x=P, ldx=40, type=BF16, codes=P, ldc=32, scales=P, lds=2)
    a.update(kw)
    return list(a.values())


def dequantize(**kw):
    a = dict(rows=4, k=40, codes=P, ldc=32, scales=P, lds=2, x=P, ldx=40, type=BF16)
    a.update(kw)
    return list(a.values())


def product(**kw):
    a = dict(groups=2, rows=4, n=8, k=40, offsets=P, index=P, rows_a=4, a=P, lda=32, sa=P, ldsa=2, b=P, ldb=32,
             stride=256, sb=P, ldsb=2, strides=16, c=P, ldc=8, ctype=BF16)
    a.update(kw)
    return list(a.values())


def logprobs(**kw):
    a = dict(rows=4, vocab=100, x=P, ld=100, type=BF16, targets=P, ttype=I64, lp=P, h=P, stats=P, top=3, tl=P, ti=P,
             buffer=P)
    a.update(kw)
    return list(a.values())


def logprobs_grad(**kw):
    a = dict(rows=4, vocab=100, x=P, ld=100, type=BF16, targets=P, ttype=I64, stats=P, h=P, top=3, ti=P, gl=P, gh=P,
             gt=P, out=P, ldo=100)
    a.update(kw)
    return list(a.values())


CASES = [
    ("aclsparseMx4Quantize", quantize, [
        (dict(rows=-1), INVALID), (dict(k=-1), INVALID), (dict(k=2**31 - 1, ldx=2**31, ldc=2**31, lds=2**31), UNSUPPORTED),
        (dict(type=I8), UNSUPPORTED), (dict(x=0), INVALID), (dict(codes=0), INVALID), (dict(scales=0), INVALID),
        (dict(ldx=39), INVALID), (dict(ldc=31), INVALID), (dict(lds=1), INVALID), (dict(rows=0), OK), (dict(k=0), OK)]),
    ("aclsparseMx4Dequantize", dequantize, [
        (dict(rows=-1), INVALID), (dict(type=I8), UNSUPPORTED), (dict(codes=0), INVALID), (dict(scales=0), INVALID),
        (dict(x=0), INVALID), (dict(ldx=39), INVALID), (dict(ldc=31), INVALID), (dict(lds=1), INVALID),
        (dict(rows=0), OK)]),
    ("aclsparseGroupedMMMx4", product, [
        (dict(groups=0), INVALID), (dict(rows=-1), INVALID), (dict(n=-1), INVALID), (dict(k=-1), INVALID),
        (dict(rows=2**31 - 64, rows_a=2**31 - 64), UNSUPPORTED), (dict(n=2**31 - 64, ldc=2**31), UNSUPPORTED),
        (dict(groups=2**31 - 64), UNSUPPORTED), (dict(offsets=0), INVALID), (dict(index=0, rows_a=3), INVALID),
        (dict(rows_a=0), INVALID), (dict(ctype=I8), UNSUPPORTED), (dict(lda=31), INVALID), (dict(ldb=16), INVALID),
        (dict(ldsa=1), INVALID), (dict(ldsb=1), INVALID), (dict(ldc=7), INVALID), (dict(stride=-16), INVALID),
        (dict(strides=-1), INVALID), (dict(c=0), INVALID), (dict(a=0), INVALID), (dict(b=0), INVALID),
        (dict(sa=0), INVALID), (dict(sb=0), INVALID), (dict(a=P + 8), INVALID), (dict(lda=40), INVALID),
        (dict(b=P + 1), INVALID), (dict(ldb=33), INVALID), (dict(stride=257), INVALID), (dict(rows=0), OK),
        (dict(n=0), OK)]),
    ("aclsparseTokenLogprobs", logprobs, [
        (dict(rows=-1), INVALID), (dict(vocab=0), INVALID), (dict(top=-1), INVALID), (dict(top=101), INVALID),
        (dict(top=65), UNSUPPORTED), (dict(vocab=2**30 + 1, ld=2**31), UNSUPPORTED), (dict(rows=2**31), UNSUPPORTED),
        (dict(type=I8), UNSUPPORTED), (dict(ttype=F32), UNSUPPORTED), (dict(ld=99), INVALID), (dict(x=0), INVALID),
        (dict(buffer=0), INVALID), (dict(targets=0), INVALID), (dict(lp=0), INVALID), (dict(tl=0), INVALID),
        (dict(ti=0), INVALID), (dict(rows=0), OK)]),
    ("aclsparseTokenLogprobsGrad", logprobs_grad, [
        (dict(rows=-1), INVALID), (dict(top=65), UNSUPPORTED), (dict(type=I8), UNSUPPORTED),
        (dict(ttype=F16), UNSUPPORTED), (dict(ld=99), INVALID), (dict(ldo=99), INVALID), (dict(x=0), INVALID),
        (dict(stats=0), INVALID), (dict(out=0), INVALID), (dict(targets=0), INVALID), (dict(h=0), INVALID),
        (dict(ti=0), INVALID), (dict(top=0), INVALID), (dict(rows=0), OK)]),
]


@pytest.mark.parametrize("name,args,changes", CASES, ids=[c[0] for c in CASES])
def test_status_codes(lib, handle, name, args, changes):
    fn = getattr(lib, name)
    assert fn(None, *args()) == Status.HANDLE_IS_NULLPTR
    for change, status in changes:
        assert fn(handle, *args(**change)) == status, (name, change)


def tensor(**kw):
    a = dict(param=P, grad=P, master=P, moments=P, exponents=None, count=10, paramType=BF16, gradType=F32)
    a.update(kw)
    return AdamWTensor(**a)


def options(**kw):
    a = dict(lr=1e-3, beta1=0.9, beta2=0.99, eps=1e-8, weightDecay=0.1, lrDevice=None, gradScale=None, step=P, buffer=P, seed=0,
             momentBits=32)
    a.update(kw)
    return AdamWOptions(**a)


def test_adamw_status_codes(lib, handle):
    def call(t, o, h=handle, count=1):
        return lib.aclsparseAdamW(h, count, ctypes.byref(t) if t else None, ctypes.byref(o) if o else None)

    assert call(tensor(), options(), None) == Status.HANDLE_IS_NULLPTR
    assert call(tensor(), None) == INVALID and call(None, options()) == INVALID
    assert call(tensor(), options(), count=-1) == INVALID
    for change, status in ((dict(beta1=1.0), INVALID), (dict(beta1=-0.1), INVALID), (dict(beta2=1.5), INVALID),
                           (dict(eps=-1.0), INVALID), (dict(eps=float("nan")), INVALID), (dict(lr=float("inf")), INVALID),
                           (dict(lr=-1.0), INVALID), (dict(weightDecay=-0.1), INVALID), (dict(step=None), INVALID), (dict(buffer=None), INVALID),
                           (dict(momentBits=16), UNSUPPORTED), (dict(momentBits=8), INVALID)):
        assert call(tensor(), options(**change)) == status, change
    for change, status in ((dict(count=-1), INVALID), (dict(paramType=I8), UNSUPPORTED),
                           (dict(gradType=I32), UNSUPPORTED), (dict(param=None), INVALID),
                           (dict(moments=None), INVALID), (dict(exponents=P), INVALID), (dict(moments=P + 2), INVALID),
                           (dict(count=2**43), UNSUPPORTED)):
        assert call(tensor(**change), options()) == status, change
    assert call(tensor(exponents=P, moments=P + 4), options(momentBits=8)) == INVALID


def test_adamw_moments_status_codes(lib, handle):
    def call(t, h=handle, count=1):
        return lib.aclsparseAdamWMoments(h, count, ctypes.byref(t) if t else None)

    assert call(tensor(), None) == Status.HANDLE_IS_NULLPTR
    assert call(None) == INVALID and call(tensor(), count=-1) == INVALID
    assert call(tensor(exponents=None)) == INVALID and call(tensor(exponents=P, master=None)) == INVALID
    assert call(tensor(exponents=P, moments=P + 4)) == INVALID and call(tensor(count=0)) == OK
    assert call(tensor(), count=0) == OK


def test_buffer_size(lib, handle):
    fn, size = lib.aclsparseTokenLogprobs_bufferSize, ctypes.c_size_t(0)
    for rows, vocab, top in ((0, 1, 0), (1, 131072, 20), (1, 2**30, 64), (37, 32003, 5), (8192, 65536, 64)):
        assert fn(handle, rows, vocab, top, ctypes.byref(size)) == OK
        # 64 records a row at most, and 1024 in all
        assert size.value % 64 == 0 and 64 <= size.value <= 1024 * (16 + 8 * top) + 64
    assert fn(handle, 1, 10, 0, None) == INVALID and fn(handle, 1, 10, 11, ctypes.byref(size)) == INVALID
    assert fn(handle, 1, 100, 65, ctypes.byref(size)) == UNSUPPORTED
    assert fn(None, 1, 10, 0, ctypes.byref(size)) == Status.HANDLE_IS_NULLPTR


# ----------------------------------------------------------------------------------------------------- the module


def mx4(*lead, blocks=2):
    return ops_sparse.MX4(torch.zeros(*lead, 16 * blocks, dtype=torch.uint8),
                          torch.zeros(*lead, blocks, dtype=torch.uint8))


def test_cpu_tensors_are_refused():
    x, t, p = torch.zeros(4, 64), torch.zeros(4, dtype=torch.int64), [torch.zeros(3)]
    for call in (lambda: ops_sparse.mx4_quantize(x), lambda: ops_sparse.mx4_dequantize(mx4(4)),
                 lambda: ops_sparse.grouped_mm_mx4(mx4(4), mx4(5)), lambda: ops_sparse.token_logprobs(x, t),
                 lambda: ops_sparse.adamw_step(p, p, ops_sparse.adamw_state(p), 1e-3),
                 lambda: ops_sparse.adamw_moments(ops_sparse.adamw_state(p, bits=8))):
        with pytest.raises(ValueError, match="ROCm device"):
            call()


def test_mx4_refusals():
    x = torch.zeros(4, 64)
    with pytest.raises(TypeError, match="float32"):
        ops_sparse.mx4_quantize(x.double())
    with pytest.raises(ValueError, match="dimension"):
        ops_sparse.mx4_quantize(x[0, 0])
    with pytest.raises(TypeError, match="uint8"):
        ops_sparse.mx4_dequantize(ops_sparse.MX4(x, mx4(4).scales))
    with pytest.raises(ValueError, match="blocks"):
        ops_sparse.mx4_dequantize(ops_sparse.MX4(mx4(4).codes[:, 1:], mx4(4).scales))
    with pytest.raises(ValueError, match="blocks"):
        ops_sparse.mx4_dequantize(ops_sparse.MX4(mx4(4).codes, mx4(5).scales))
    for width in (32, 65, 0, -1):
        with pytest.raises(ValueError, match="width"):
            ops_sparse.mx4_dequantize(mx4(4), width)
    with pytest.raises(TypeError, match="dtype"):
        ops_sparse.mx4_dequantize(mx4(4), dtype=torch.float64)
    with pytest.raises(ValueError, match="gather"):
        ops_sparse.grouped_mm_mx4(mx4(4), mx4(5), gather=True)
    with pytest.raises(ValueError, match=r"\[N, K\]"):
        ops_sparse.grouped_mm_mx4(mx4(4), mx4(2, 5))
    with pytest.raises(ValueError, match="codes of"):
        ops_sparse.grouped_mm_mx4(mx4(4), mx4(5, blocks=3))
    with pytest.raises(TypeError, match="out_dtype"):
        ops_sparse.grouped_mm_mx4(mx4(4), mx4(5), out_dtype=torch.int8)


def test_logprobs_refusals():
    x, t = torch.zeros(4, 64), torch.zeros(4, dtype=torch.int64)
    for bad in ((x, t[:3]), (x, t.view(2, 2)), (x[0], t)):
        with pytest.raises(ValueError, match="targets"):
            ops_sparse.token_logprobs(*bad)
    with pytest.raises(TypeError, match="logits"):
        ops_sparse.token_logprobs(x.double(), t)
    with pytest.raises(TypeError, match="targets"):
        ops_sparse.token_logprobs(x, t.float())
    with pytest.raises(ValueError, match="vocabulary"):
        ops_sparse.token_logprobs(x[:, :0], t)
    for top in (-1, 65, 100):
        with pytest.raises(ValueError, match="top"):
            ops_sparse.token_logprobs(x, t, top=top)
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="forward"):
            ops_sparse.token_logprobs(torch.autograd.forward_ad.make_dual(x, x), t)
        with pytest.raises(NotImplementedError, match="forward"):
            ops_sparse.mx4_quantize(torch.autograd.forward_ad.make_dual(x, x))


def test_adamw_state():
    params = [torch.randn(3, 5), torch.randn(64).bfloat16(), torch.randn(0)]
    state = ops_sparse.adamw_state(params, bits=8, seed=5)
    assert [m.shape for m in state.moments] == [(2, 32), (2, 64), (2, 0)]
    assert [e.shape for e in state.exponents] == [(2, 1), (2, 2), (2, 0)]
    assert all(m.dtype == torch.uint8 for m in state.moments + state.exponents) and state.seed == 5
    assert all(torch.equal(m, p.float()) and m.data_ptr() != p.data_ptr() or p.numel() == 0
               for m, p in zip(state.masters, params))
    state = ops_sparse.adamw_state([p.float() for p in params])
    assert state.exponents is None and state.masters is None and state.step.tolist() == [0, 0]
    assert all(m.dtype == torch.float32 for m in ops_sparse.adamw_moments(state))
    assert ops_sparse.adamw_state(params, masters=False).masters is None
    with pytest.raises(ValueError, match="bits"):
        ops_sparse.adamw_state(params, bits=16)
    with pytest.raises(ValueError, match="parameter"):
        ops_sparse.adamw_state([])


def test_random_bits_are_even_and_independent():
    # of n numbers each bit is set n / 2 times and agrees with another number's as often, both within 5 deviations,
    # sqrt(n) / 2 each: between neighbours, steps, tensors, seeds and the two halves
    from test_gpu_adamw import random_bits

    n = 1 << 16
    base = random_bits(n, 7, 100, 3)
    others = [np.roll(base, 1), np.roll(base, 32), base >> np.uint64(16), random_bits(n, 8, 100, 3),
              random_bits(n, 7, 101, 3), random_bits(n, 7, 100, 4)]
    limit = 5 * n**0.5 / 2
    for i in range(32):
        bit = (base >> np.uint64(i)) & np.uint64(1)
        assert abs(int(bit.sum()) - n / 2) <= limit
        for j, other in enumerate(others):
            if j == 2 and i >= 16:
                continue
            same = bit == ((other >> np.uint64(i)) & np.uint64(1))
            assert abs(int(same.sum()) - n / 2) <= limit, (i, j)


def test_the_copies_to_lds_are_the_only_use_of_m0(tmp_path):
    # the 4-bit products' tiles set m0 in assembly that cannot say so, as the other grouped products do
    from test_experts_abi import other_uses_of_m0

    tool = "/opt/rocm/llvm/bin/llvm-objdump"
    shutil.copy(_lib.LIB_PATH, tmp_path / "lib.so")
    subprocess.run([tool, "--offloading", "lib.so"], cwd=tmp_path, check=True, capture_output=True)
    images = [f for f in tmp_path.iterdir() if f.name.endswith("gfx950") and b"Mx4TileKernel" in f.read_bytes()]
    assert len(images) == 1
    text = subprocess.run([tool, "-d", "--no-show-raw-insn", images[0].name], cwd=tmp_path, check=True,
                          capture_output=True, text=True).stdout
    lines = [line.split("//")[0].strip() for line in text.splitlines()]
    assert sum(line.startswith("global_load_lds_dwordx4 ") for line in lines) > 100
    assert other_uses_of_m0(lines) == []


def test_scaled_products_in_assembly_follow_their_wait(tmp_path):
    # a matrix instruction written as assembly has the wait for what an ordinary instruction wrote right before it
    tool = "/opt/rocm/llvm/bin/llvm-objdump"
    shutil.copy(_lib.LIB_PATH, tmp_path / "lib.so")
    subprocess.run([tool, "--offloading", "lib.so"], cwd=tmp_path, check=True, capture_output=True)
    image = next(f for f in tmp_path.iterdir() if f.name.endswith("gfx950") and b"Mx4TileKernel" in f.read_bytes())
    text = subprocess.run([tool, "-d", "--no-show-raw-insn", image.name], cwd=tmp_path, check=True, capture_output=True,
                          text=True).stdout
    kernel, count = "", 0
    lines = [line.split("//")[0].strip() for line in text.splitlines()]
    for before, line in zip(lines, lines[1:]):
        if line.endswith(">:"):
            kernel = line
        if "TileKernel" in kernel and line.startswith("v_mfma_scale"):
            count += 1
            assert before == "s_nop 1"
    assert count > 1000


def test_factors_are_odd_numbers_of_32_bits(lib, handle):
    for first, second in ((2, 3), (3, 0)):
        assert lib.aclsparseAdamWMixed(handle, 1, ctypes.byref(tensor()), ctypes.byref(options()), first, second) == INVALID
    assert lib.aclsparseAdamWMixed(None, 0, None, None, 3, 5) == Status.HANDLE_IS_NULLPTR
    p = [torch.zeros(3)]
    state = ops_sparse.adamw_state(p, bits=8)
    assert state.factors is None
    for factors in ((2, 3), (3, 2**32 + 1), (-1, 3)):
        with pytest.raises(ValueError, match="factors"):
            ops_sparse.adamw_step(p, p, state._replace(factors=factors), 1e-3)
    with pytest.raises(ValueError, match="ROCm device"):
        ops_sparse.adamw_step(p, p, state._replace(factors=(3, 5)), 1e-3)


def test_which_kernel_multiplies(lib):
    # the rule of the 4-bit products, an internal function of the library, for the shapes that the GPU tests name
    import test_gpu_mx4 as gpu

    rule = getattr(lib, "_ZN5aclsp11Mx4KernelOfElllll")
    rule.argtypes, rule.restype = [ctypes.c_int64] * 5, ctypes.c_int

    def kernel(groups, rows, n, k):
        return gpu.KERNELS[rule(groups, rows, n, (k + 31) // 32, 256)]

    for name, lens, n, k in gpu.REACHED:
        assert kernel(len(lens), sum(lens), n, k) == name, (lens, n, k)
    assert {c[0] for c in gpu.REACHED} == set(gpu.KERNELS)
    for name, lens, n, k in gpu.NO_EXPERT:
        assert kernel(len(lens), sum(lens) + 14, n, k) == name, (lens, n, k)
    for name, tokens, experts, chosen, n, k in gpu.GATHERED:
        assert kernel(experts, tokens * chosen, n, k) == name, (tokens, n, k)
    assert kernel(2, 3300, 2048, 290) == kernel(2, 3300, 2048, 520) == kernel(3, 3400, 2048, 300) == "256x256"
    # and those that the first tests took for large tiles reach the small ones
    assert kernel(1, 2500, 2048, 288) == kernel(4, 2900, 700, 520) == "64x128"


def test_width_of_rows_of_no_blocks():
    for width in (-1, -31, 1):
        with pytest.raises(ValueError, match="width"):
            ops_sparse.mx4_dequantize(mx4(4, blocks=0), width)
    with pytest.raises(ValueError, match="ROCm device"):
        ops_sparse.mx4_dequantize(mx4(4, blocks=0), 0)


def test_a_gradient_in_the_logits_place_has_their_rows(lib, handle):
    grad = lib.aclsparseTokenLogprobsGrad
    assert grad(handle, *logprobs_grad(ldo=101)) == INVALID and grad(handle, *logprobs_grad(ld=101)) == INVALID
    assert grad(handle, *logprobs_grad(ldo=101, rows=0)) == OK
