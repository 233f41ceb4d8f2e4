"""The quantised linear layer's buffers on the GPU: strided, shared and
pitched ones."""
import numpy as np
import pytest
import torch

import linear_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ody():
    import odyssey_b200
    odyssey_b200.lib()
    return odyssey_b200


def test_strided_host_weight(ody):
    """Every other byte of a buffer as the weight, in numpy and in torch."""
    rng = np.random.default_rng(1)
    out, inn = 1024, 1024
    q = R.random_weight(rng, R.NVFP4, out, inn)
    wide = rng.integers(0, 256, 2 * q.size, dtype=np.uint8)
    wide[::2] = q
    x = rng.standard_normal((3, 1024)).astype(np.float32)
    for fn in (ody.fp4_linear, ody.fp4_linear_dgrad):
        want = fn(x, ody.QuantizedTensor(q, R.NVFP4, out * inn))
        assert np.array_equal(fn(x, ody.QuantizedTensor(wide[::2], R.NVFP4, out * inn)), want)
        strided = ody.QuantizedTensor(torch.from_numpy(wide)[::2], R.NVFP4, out * inn)
        assert np.array_equal(fn(torch.from_numpy(x), strided).numpy(), want)


def test_host_results_over_their_operands(ody):
    """A host call of the stateless operations whose result takes an operand's
    place gives the result, not the operand."""
    from odyssey_b200 import _lib as L
    lib = L.lib()
    rng = np.random.default_rng(2)
    g, p, m, v = (rng.standard_normal(1000).astype(np.float32) for _ in range(4))
    v = np.abs(v)
    apart, over = np.empty_like(g), g.copy()
    L.check(lib.ody_unscale(g.ctypes.data, L.F32, 1000, 3.0, apart.ctypes.data))
    L.check(lib.ody_unscale(over.ctypes.data, L.F32, 1000, 3.0, over.ctypes.data))
    assert np.array_equal(over, apart) and not np.array_equal(over, g)
    want = ody.adamw_step(p, g, m, v, 1, 1e-3)
    args = [a.ctypes.data for a in (p, g, m, v)]
    L.check(lib.ody_adamw_step(*args, 1000, 1, 1e-3, 0.9, 0.999, 1e-8, 0.01, args[0], args[2], args[3]))
    for got, w in zip((p, m, v), want):
        assert np.array_equal(got, w)


def test_device_results_that_overlap_operands_are_refused(ody):
    """A result that shares a byte with an operand is turned away; columns of
    one buffer that lie between the operand's are not."""
    from odyssey_b200 import _lib as L
    lib = L.lib()
    st = torch.cuda.current_stream().cuda_stream
    rng = np.random.default_rng(3)
    out, inn, rows, ld = 32, 64, 6, 200
    q = torch.from_numpy(R.random_weight(rng, R.NVFP4, out, inn)).cuda()
    w = ody.QuantizedTensor(q, R.NVFP4, out * inn)
    buf = torch.randn(3 * rows, ld, device="cuda")
    before = buf.clone()

    def call(y, ldy, x=(0, 0), ldx=ld, n=rows, q=q.data_ptr(), ts=None):
        at = lambda p: buf.data_ptr() + 4 * (p[0] * ld + p[1])
        return lib.ody_fp4_linear_on_stream(R.NVFP4, q, ts, 1.0, out, inn, at(x), L.F32, n, ldx, at(y), L.F32, ldy, None, 0, st)

    for y, ldy in (((0, 0), ld), ((0, 63), ld), ((0, ld - 31), ld), ((rows - 1, 63), ld), ((rows - 1, 10), 2 * ld),
                   ((0, 64), ld - 1), ((0, 100), 130), ((0, 150), 2 * ld + 49)):
        x = (1, 0) if y == (0, ld - 31) else (0, 0)  # there y's rows end in the first column of x's next ones
        assert call(y, ldy, x) == L.ERR_ARG, (y, ldy)
    whole = ody.QuantizedTensor(buf.view(torch.uint8).view(-1)[:q.numel()], R.NVFP4, out * inn)
    assert call((0, 60), ld, (rows, 0), q=whole.data.data_ptr()) == L.ERR_ARG
    assert call((0, 0), ld, (rows, 0), ts=buf.data_ptr() + 4 * ld) == L.ERR_ARG
    torch.cuda.synchronize()
    assert torch.equal(buf, before)
    for y, ldy, x in (((0, 64), ld, (0, 0)), ((0, ld - 32), ld, (1, 0)), ((0, 64), 2 * ld, (1, 0)), ((rows, 0), ld, (0, 0)), ((rows, 0), 32, (0, 0))):
        want = ody.fp4_linear(buf[x[0]:x[0] + rows, :inn].clone(), w)
        assert call(y, ldy, x) == L.OK
        got = torch.as_strided(buf, (rows, out), (ldy, 1), y[0] * ld + y[1])
        assert torch.equal(got, want)
        buf.copy_(before)
    # through Python: a view of the input's memory, and of the activation's
    x = torch.randn(8, 64, device="cuda")
    for o in (x.view(-1)[:8 * 32].view(8, 32), x.view(-1)[64:64 + 8 * 32].view(8, 32), x.view(-1)[256:].view(8, 32)):
        with pytest.raises(ody.OdysseyError, match="overlap an operand"):
            ody.fp4_linear(x, w, out=o)
    big = torch.zeros(4096, dtype=torch.uint8, device="cuda")
    a = ody.Activation8(big[:512].view(8, 64), torch.full((8, 2), 127, dtype=torch.uint8, device="cuda"), 8, 64)
    for at in (0, 256, 508):
        with pytest.raises(ody.OdysseyError, match="overlap an operand"):
            ody.load_activation8(a, "float32", out=big[at:at + 2048].view(torch.float32).view(8, 64))
    ody.load_activation8(a, "float32", out=big[512:2560].view(torch.float32).view(8, 64))
    with pytest.raises(ody.OdysseyError, match="overlap an operand"):
        ody.linear_wgrad8(x[:, :4].contiguous(), a, out=big[508:1020].view(torch.bfloat16).view(4, 64), out_dtype="bfloat16")
    dy = torch.randn(8, 32, device="cuda")
    acc = torch.randn(33, 64, device="cuda")
    with pytest.raises(ody.OdysseyError, match="overlap an operand"):
        ody.linear_wgrad8(dy, a, add=acc[:32], out=acc[1:])
    want = ody.linear_wgrad8(dy, a, add=acc[:32].clone())
    assert torch.equal(ody.linear_wgrad8(dy, a, add=acc[:32], out=acc[:32]), want)


def run_python(code):
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip().endswith("done"), r.stdout + r.stderr


LAYERS = """
import ctypes as C, threading, torch, odyssey_b200 as ody
def layer(kind, block, size, out, inn, rows, dtype):
    g = torch.Generator(device="cuda").manual_seed(out)
    q = torch.randint(0, 120, (out * inn // block * size,), dtype=torch.uint8, device="cuda", generator=g)
    return ody.QuantizedTensor(q, kind, out * inn), torch.randn(rows, out, device="cuda", generator=g).to(dtype)
"""


def test_shared_memory_limit_is_one_number(ody):
    """A few-row backward product over a long reduction takes more shared
    memory than one over a short one.  What a kernel may take does not depend
    on which came first, so threads that set it cross without harm."""
    run_python(LAYERS + """
def limit():
    n = C.c_int32(0)
    assert ody.lib().odyx_linear_rows_limit(C.byref(n)) == 0
    return n.value
w, dy = layer(6, 32, 17, 64, 64, 1, torch.bfloat16)
ody.fp4_linear_dgrad(dy, w)
short = limit()
w, dy = layer(6, 32, 17, 70000, 64, 1, torch.bfloat16)
ody.fp4_linear_dgrad(dy, w)
torch.cuda.synchronize()
assert short == limit(), (short, limit())
print("done")
""")


def test_first_calls_from_threads_at_once(ody):
    """A process's first calls of every kind and type, short and long
    reductions at once from two threads each (four in all), give what later calls give."""
    run_python(LAYERS + """
errors, results = [], []
for kind, block, size in ((6, 32, 17), (7, 16, 9), (9, 32, 17)):
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        for rows in (1, 4, 300):
            sets = [layer(kind, block, size, out, inn, rows, dtype) for out, inn in ((64, 64), (20000, 64))] * 2
            torch.cuda.synchronize()
            start, got = threading.Barrier(len(sets)), [None] * len(sets)
            def call(i):
                try:
                    start.wait()
                    with torch.cuda.stream(torch.cuda.Stream()):
                        got[i] = (ody.fp4_linear_dgrad(sets[i][1], sets[i][0]),)
                        torch.cuda.current_stream().synchronize()
                except Exception as e:
                    errors.append(repr(e))
            ts = [threading.Thread(target=call, args=(i,)) for i in range(len(sets))]
            [t.start() for t in ts]
            [t.join() for t in ts]
            assert not errors, errors
            for (w, dy), (y,) in zip(sets, got):
                assert torch.equal(ody.fp4_linear_dgrad(dy, w), y)
torch.cuda.synchronize()
print("done")
""")


def test_few_rows_take_no_workspace(ody):
    """NVFP4 with a width of 16s that is not one of 32s: the call brings none
    and allocates nothing but its result."""
    from odyssey_b200 import _lib as L
    rng = np.random.default_rng(4)
    out, inn = 4096, 4080
    q = R.random_weight(rng, R.NVFP4, out, inn)
    w = ody.QuantizedTensor(torch.from_numpy(q).cuda(), R.NVFP4, out * inn)
    w64 = R.weight(R.NVFP4, q, out, inn)
    for rows, op, fn, cols, others, m in ((8, L.LINEAR_FORWARD, ody.fp4_linear, inn, out, w64.T),
                                          (4, L.LINEAR_DGRAD, ody.fp4_linear_dgrad, out, inn, w64)):
        x = torch.from_numpy(rng.standard_normal((rows, cols)).astype(np.float32)).cuda()
        x64 = R.to64(x)
        fn(x, w)  # loads the kernels
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        y = fn(x, w)
        assert torch.cuda.max_memory_allocated() - before < 2 * 4 * rows * others
        R.check(y, x64 @ m, R.tolerance(np.abs(x64) @ np.abs(m), cols, x64 @ m, "float32"))
        z = torch.empty_like(y)
        entry = L.lib().ody_fp4_linear_on_stream if op == L.LINEAR_FORWARD else L.lib().ody_fp4_linear_dgrad_on_stream
        assert entry(w.kind, w.data.data_ptr(), None, 1.0, out, inn, x.data_ptr(), L.F32, rows, cols, z.data_ptr(), L.F32,
                     others, None, 0, torch.cuda.current_stream().cuda_stream) == L.OK
        assert torch.equal(z, y)


HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def check_gemm(got, terms, reduction, want):
    """Bound on the tcgen05 path's error with bfloat16 operands, whose products
    are exact.  One mma adds 16 of them and what the accumulator holds, each
    cut off at 2^-24 of the largest or below: 17 x 2^-24 of the magnitudes'
    sum `terms`.  An accumulator takes 32 mma (64 where the result has 16
    bits), so all of them together lose at most that many times as much of
    all terms.  The accumulators, one per 512 (1024) of the reduction, and a
    shared tile's pieces (sqrt(steps) / 2 + 2 at most, steps of 64) are added
    with rounding; two roundings of the scale and half a step of the result
    follow."""
    half = HALF_STEP[got.dtype]
    mma, chunk = (32, 512) if got.dtype == torch.float32 else (64, 1024)
    adds = reduction / chunk + 1 + (reduction / 64) ** 0.5 / 2 + 2
    tol = terms * (mma * 17 * 2.0 ** -24 + adds * 2.0 ** -24 + 2.0 ** -23)
    R.check(got, want, tol + (np.abs(want) + tol) * half)


def pitched(rng, rows, cols, pitch, start=8):
    """bfloat16 rows whose begin and pitch are multiples of 16 bytes, NaN all around."""
    buf = torch.full((rows + 2, pitch), float("nan"), dtype=torch.bfloat16, device="cuda")
    view = buf[1:rows + 1, start:start + cols]
    view.copy_(torch.from_numpy(rng.standard_normal((rows, cols)).astype(np.float32)))
    assert view.data_ptr() % 16 == 0 and pitch % 8 == 0 and pitch > start + cols
    return view


@pytest.mark.parametrize("rows,out,inn", [(700, 1100, 1030), (1025, 769, 1568), (300, 2500, 2000), (257, 3001, 4112)])
@pytest.mark.parametrize("out_dtype", ["bfloat16", "float32"])
def test_rows_read_in_place_at_a_pitch(ody, rows, out, inn, out_dtype):
    """bfloat16 rows that the tensor map reads where they lie, wider apart than
    their columns (whole and broken eights and tiles): nothing of what lies
    around them reaches a result."""
    from odyssey_b200 import _lib as L
    rng = np.random.default_rng(rows)
    of = L.lib().ody_linear_workspace_of
    assert all(of(op, 6 * (op < 2), rows, out, inn, L.BF16) > 0 for op in range(3))  # none: another path
    q = R.random_weight(rng, R.MXFP4, out, inn)
    w, w64 = ody.QuantizedTensor(torch.from_numpy(q).cuda(), R.MXFP4, out * inn), R.weight(R.MXFP4, q, out, inn)
    for fn, cols, m in ((ody.fp4_linear, inn, w64.T), (ody.fp4_linear_dgrad, out, w64)):
        x = pitched(rng, rows, cols, (cols + 31) // 8 * 8)
        x64 = R.to64(x)
        check_gemm(fn(x, w, out_dtype=out_dtype), np.abs(x64) @ np.abs(m), cols, x64 @ m)
        assert torch.equal(fn(x, w, out_dtype=out_dtype), fn(x.contiguous(), w, out_dtype=out_dtype))
    a = ody.save_activation8(pitched(rng, rows, inn, (inn + 31) // 8 * 8))
    dy = pitched(rng, rows, out, (out + 31) // 8 * 8, 16)
    d64, x64 = R.to64(dy), R.to64(ody.load_activation8(a, "float32"))
    check_gemm(ody.linear_wgrad8(dy, a, out_dtype=out_dtype), np.abs(d64.T) @ np.abs(x64), rows, d64.T @ x64)
