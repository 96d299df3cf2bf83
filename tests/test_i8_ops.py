"""8-bit rows (gann_quantize_rows) and their products (gann_matmul_i8) against
exact arithmetic in 64 bits."""
import ctypes as C
import threading

import numpy as np
import pytest
import torch

from gustann_b200 import api
from gustann_b200.api import GustANNError, matmul_i8, quantize_rows

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODE = {"f32": api.F32, "f16": api.F16, "bf16": api.BF16}


def ref_quantize(x):
    """Codes and scales of float rows; the quotient in 64 bits, where x / scale
    of two float32 values is never mistaken for a tie."""
    x = x.float().cpu().numpy()
    amax = np.abs(x).max(1)
    with np.errstate(all="ignore"):
        scale = np.where(np.isfinite(amax), amax * (np.float32(1) / np.float32(127)), np.float32(np.nan)).astype(np.float32)
        q = np.rint(x.astype(np.float64) / scale.astype(np.float64)[:, None])
    live = (scale > 0)[:, None]
    return np.where(live, np.clip(q, -127, 127), 0).astype(np.int8), scale


def check_quantize(x):
    codes, scales = quantize_rows(x)
    rc, rs = ref_quantize(x)
    assert codes.shape == x.shape and (codes.shape[0] < 2 or codes.stride(0) % 16 == 0)
    assert np.array_equal(scales.cpu().numpy(), rs, equal_nan=True)
    assert np.array_equal(codes.cpu().numpy(), rc)


def i8(rows, cols, seed, room=0):
    """Random codes, -128 among them, in rows of 16-byte multiples (+ room)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    stride = (cols + 15) // 16 * 16 + 16 * room
    full = torch.randint(-128, 128, (rows, stride), generator=g, device="cuda", dtype=torch.int8)
    s = torch.rand(rows, generator=g, device="cuda") * 0.02 + 1e-3
    return full[:, :cols], s


def check_matmul(y, a, sa, b, sb, bias):
    """The sum is exact; its conversion to float32, the product with sa and the
    last fused step each round by half a step of float32 (2^-24 relative), the
    output by half a step of its type."""
    t = (a.cpu().double() @ b.cpu().double().T) * sa.cpu().double()[:, None] * sb.cpu().double()[None, :]
    ref = t + bias.cpu().double() if bias is not None else t
    half = torch.finfo(y.dtype).eps / 2 if y.dtype != torch.float32 else 0.0
    tiny = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}[y.dtype]
    bound = 1.01 * (2 * 2.0 ** -24 * t.abs() + (2.0 ** -24 + half) * ref.abs()) + tiny
    err = (y.cpu().double() - ref).abs()
    over = ref.abs() > torch.finfo(y.dtype).max * (1 - half)      # beyond the type: infinite is right
    assert bool(((err <= bound) | over).all()), float((err - bound).max())


# ------------------------------------------------------------------ quantize
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("rows,dim", [(1, 1), (1, 768), (7, 15), (61, 16), (33, 100), (130, 768), (5, 1023), (3, 4096),
                                      (2, 20001), (1, 131071), (5000, 33), (70000, 8)])
def test_quantize_equals_exact(rows, dim, dtype):
    g = torch.Generator(device="cuda").manual_seed(rows * 7 + dim)
    x = torch.randn(rows, dim, generator=g, device="cuda") * torch.rand(rows, 1, generator=g, device="cuda")
    x[rows // 2:rows // 2 + 1] = 0
    check_quantize(x.to(DT[dtype]))


@pytest.mark.gpu
def test_quantize_ties_and_extremes():
    # scale 1: halves are ties, which go to the even code
    x = torch.tensor([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5, -126.5, 126.5, 125.5, 0.49999997, 0.50000006]], device="cuda")
    codes, scales = quantize_rows(x)
    assert scales.tolist() == [1.0]
    assert codes.tolist() == [[127, 0, 2, 2, 0, -2, -126, 126, 126, 0, 1]]
    # many quotients beside a tie, at many scales
    g = torch.Generator(device="cuda").manual_seed(5)
    s = torch.rand(4096, 1, generator=g, device="cuda") + 0.5
    n = torch.randint(-126, 127, (4096, 64), generator=g, device="cuda").float() + 0.5
    y = (n * s).contiguous()
    y.view(torch.int32).add_(torch.randint(-1, 2, y.shape, generator=g, device="cuda", dtype=torch.int32))
    y[:, 0:1] = 127 * s
    check_quantize(y)
    # tiny and huge rows: a scale below float32's normal range, one that is zero
    rows = [torch.full((9,), v, device="cuda") * torch.linspace(-1, 1, 9, device="cuda")
            for v in (3.4e38, 1e30, 1e-30, 1e-36, 3e-38, 1e-40, 2e-43, 9e-44, 1e-45)]
    check_quantize(torch.stack(rows))


@pytest.mark.gpu
def test_quantize_bad_rows_and_layouts():
    x = torch.randn(6, 40, device="cuda")
    x[1, 39] = float("nan")
    x[2, 0] = float("inf")
    x[3, 7] = -float("inf")
    check_quantize(x)
    codes, scales = quantize_rows(x)
    assert torch.isnan(scales).tolist() == [False, True, True, True, False, False]
    assert not codes[1:4].any()
    # strided, unaligned and repeated rows
    for dt in DT.values():
        big = torch.randn(50, 131, device="cuda").to(dt)
        check_quantize(big[:, 1:100])
        check_quantize(big[::3, 2:131])
        check_quantize(big[:1].expand(20, 131))
    assert quantize_rows(x[:0])[0].shape == (0, 40)


@pytest.mark.gpu
def test_quantize_leaves_the_rest_of_a_row():
    x = torch.randn(37, 70, device="cuda")
    buf = torch.full((37, 96), 99, dtype=torch.int8, device="cuda")
    s = torch.empty(37, device="cuda")
    api._check(api.lib.gann_quantize_rows(x.data_ptr(), 37, 280, 70, api.F32, buf.data_ptr(), 96, s.data_ptr(), 0,
                                          torch.cuda.current_stream().cuda_stream or None))
    assert bool((buf[:, 70:] == 99).all())
    assert np.array_equal(buf[:, :70].cpu().numpy(), ref_quantize(x)[0])


# -------------------------------------------------------------------- matmul
SHAPES = [(1, 1, 1), (1, 17, 16), (1, 1000, 768), (2, 129, 100), (3, 4096, 512), (5, 300, 33), (8, 2049, 1024),
          (9, 128, 64), (16, 515, 2000), (17, 1000, 768), (24, 4001, 1024), (33, 128, 128), (64, 1024, 4096),
          (65, 257, 129), (100, 5001, 31), (128, 128, 128), (129, 513, 640), (257, 1025, 769), (500, 700, 100),
          (1024, 2048, 256), (2100, 130, 4097), (130, 19000, 48), (20000, 5, 300), (300, 2, 20000)]


@pytest.mark.gpu
@pytest.mark.parametrize("out", list(DT))
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_matmul_within_its_roundings(m, n, k, out):
    a, sa = i8(m, k, m + 1, room=m % 2)
    b, sb = i8(n, k, n + 2, room=n % 3)
    if out == "f16":
        sa = sa * 0.01
    bias = torch.randn(n, device="cuda") if (m + n + k) % 2 else None
    y = matmul_i8(a, sa, b, sb, bias=bias, dtype=DT[out])
    assert y.shape == (m, n) and y.dtype == DT[out]
    check_matmul(y, a, sa, b, sb, bias)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n", [(1, 3), (20, 200), (300, 300)])
def test_matmul_largest_sums_do_not_overflow(m, n):
    k = 131071
    a = torch.full((m, k + 1), -128, dtype=torch.int8, device="cuda")[:, :k]
    b = torch.full((n, k + 1), -128, dtype=torch.int8, device="cuda")[:, :k]
    one = torch.ones(max(m, n), device="cuda")
    y = matmul_i8(a, one[:m], b, one[:n])
    # 16384 * 131071 = 2^31 - 2^14 has 17 significant bits: exact in float32
    assert bool((y == float(16384 * k)).all())


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(3, 50, 64), (40, 77, 96), (300, 333, 200)])
def test_matmul_target_rows(m, n, k):
    a, sa = i8(m, k, 1)
    b, sb = i8(n, k, 2)
    want = matmul_i8(a, sa, b, sb)
    for dt in DT.values():
        for off, room in ((0, 0), (1, 3), (8, 8)):
            buf = torch.full((m + 1, n + off + room), 7.0, device="cuda", dtype=dt)
            got = matmul_i8(a, sa, b, sb, out=buf[:m, off:off + n])
            assert torch.equal(got, want.to(dt))
            assert bool((buf[m] == 7).all() and (buf[:, :off] == 7).all() and (buf[:, off + n:] == 7).all())


@pytest.mark.gpu
def test_matmul_scales_that_are_not_finite():
    a, sa = i8(40, 96, 1)
    b, sb = i8(70, 96, 2)
    sa[3], sb[5] = float("nan"), float("inf")
    sb[6] = 0
    y = matmul_i8(a, sa, b, sb, bias=torch.ones(70, device="cuda")).cpu()
    assert bool(torch.isnan(y[3]).all())
    assert bool((~torch.isfinite(y[:, 5])).all())
    assert bool((torch.cat([y[:3, 6], y[4:, 6]]) == 1).all())


@pytest.mark.gpu
def test_matmul_empty():
    a, sa = i8(4, 32, 1)
    b, sb = i8(5, 32, 2)
    assert matmul_i8(a[:0], sa[:0], b, sb).shape == (0, 5)
    assert matmul_i8(a, sa, b[:0], sb[:0]).shape == (4, 0)


@pytest.mark.gpu
def test_output_offsets_past_32_bits():
    """Rows of the output more than 2^31 elements from its start."""
    n, k, m = 70000, 32, 31000
    a, sa = i8(m, k, 1)
    b, sb = i8(n, k, 2)
    y = matmul_i8(a, sa, b, sb, dtype=torch.bfloat16)
    assert y.numel() > 2 ** 31
    check_matmul(y[-3:], a[-3:], sa[-3:], b, sb, None)
    check_matmul(y[:2], a[:2], sa[:2], b, sb, None)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(1024, 20000, 64), (600, 30000, 200), (16, 600, 4096), (200, 300, 8192)])
def test_calls_at_the_same_time(m, n, k):
    """Large products with a short k, and split ones, on four streams at once:
    blocks that work in clusters do not wait for each other's SMs."""
    a, sa = i8(m, k, 1)
    b, sb = i8(n, k, 2)
    want = matmul_i8(a, sa, b, sb, dtype=torch.bfloat16)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    outs = []
    for _ in range(6):
        for st in streams:
            with torch.cuda.stream(st):
                outs.append(matmul_i8(a, sa, b, sb, dtype=torch.bfloat16))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 40])
def test_first_cuda_call_of_a_thread(m):
    """A host thread that has made no CUDA call before calls the C entry."""
    a, sa = i8(m, 64, 1)
    b, sb = i8(70, 64, 2)
    want = matmul_i8(a, sa, b, sb)
    got = torch.zeros_like(want)
    args = (a.data_ptr(), m, 64, sa.data_ptr(), b.data_ptr(), 70, 64, sb.data_ptr(), None, 64, got.data_ptr(), 70,
            api.F32, 0, None)
    torch.cuda.synchronize()
    code = []
    t = threading.Thread(target=lambda: code.append(api.lib.gann_matmul_i8(*args)))
    t.start()
    t.join()
    torch.cuda.synchronize()
    assert code == [api.GANN_OK] and torch.equal(got, want)


@pytest.mark.gpu
def test_products_of_different_sizes_from_several_threads():
    """Plans with little and with much shared memory, launched by four threads
    at once (the library is called without the interpreter's lock)."""
    work = []
    for m, n, k in ((16, 300, 33), (16, 600, 4096), (100, 3000, 512), (8, 200, 64)):
        a, sa = i8(m, k, 1)
        b, sb = i8(n, k, 2)
        want = matmul_i8(a, sa, b, sb)
        got = torch.empty_like(want)
        args = (a.data_ptr(), m, a.stride(0), sa.data_ptr(), b.data_ptr(), n, b.stride(0), sb.data_ptr(), None, k,
                got.data_ptr(), n, api.F32, 0, torch.cuda.Stream().cuda_stream)
        work.append((args, got, want, a, sa, b, sb))
    torch.cuda.synchronize()
    start, errors = threading.Barrier(4), []

    def run(args, *_):
        start.wait()
        for _ in range(5000):
            if api.lib.gann_matmul_i8(*args):
                errors.append(api.lib.gann_last_error())
                return
    threads = [threading.Thread(target=run, args=w) for w in work]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert errors == []
    assert all(torch.equal(w[1], w[2]) for w in work)


class _KernelNode(C.Structure):
    """CUDA_KERNEL_NODE_PARAMS (v2) of the driver's API."""

    _fields_ = [("func", C.c_void_p), ("grid", C.c_uint * 3), ("block", C.c_uint * 3), ("shared", C.c_uint),
                ("params", C.c_void_p), ("extra", C.c_void_p), ("kern", C.c_void_p), ("ctx", C.c_void_p)]


def launches(call):
    """(cluster size, shared memory of a block) of the kernels that a call
    launches, read from a captured graph."""
    cu = C.CDLL("libcuda.so.1")
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        call()
    raw, n, found = C.c_void_p(graph.raw_cuda_graph()), C.c_size_t(), []
    assert cu.cuGraphGetNodes(raw, None, C.byref(n)) == 0
    nodes = (C.c_void_p * n.value)()
    assert cu.cuGraphGetNodes(raw, nodes, C.byref(n)) == 0
    for node in map(C.c_void_p, nodes):
        kind, p, cluster, static = C.c_int(), _KernelNode(), (C.c_uint * 16)(), C.c_int()
        assert cu.cuGraphNodeGetType(node, C.byref(kind)) == 0
        if kind.value:     # CU_GRAPH_NODE_TYPE_KERNEL is 0
            continue
        assert cu.cuGraphKernelNodeGetParams_v2(node, C.byref(p)) == 0
        assert cu.cuGraphKernelNodeGetAttribute(node, 4, cluster) == 0      # CU_LAUNCH_ATTRIBUTE_CLUSTER_DIMENSION
        if p.func:         # CU_FUNC_ATTRIBUTE_SHARED_SIZE_BYTES
            assert cu.cuFuncGetAttribute(C.byref(static), 1, C.c_void_p(p.func)) == 0
        else:
            assert cu.cuKernelGetAttribute(C.byref(static), 1, C.c_void_p(p.kern), 0) == 0
        found.append((max(cluster[0], 1), p.shared + static.value))
    return found


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k,size", [(16, 600, 4096, 0), (64, 200, 8192, 0), (1024, 20000, 64, 2), (600, 30000, 200, 2),
                                        (24, 32001, 1024, 1), (100, 300, 64, 1)])
def test_clusters_have_their_multiprocessors_to_themselves(m, n, k, size):
    """Blocks of a cluster need tensor memory all at once, so no block that might
    hold some, of whatever kernel, may lie beside them: their shared memory
    leaves less than the 1024 bytes that every block is charged."""
    a, sa = i8(m, k, 1)
    b, sb = i8(n, k, 2)
    matmul_i8(a, sa, b, sb)
    (cluster, shared), = launches(lambda: matmul_i8(a, sa, b, sb))
    assert cluster == size or (size == 0 and cluster > 1)      # 0: split along k
    whole = torch.cuda.get_device_properties(0).shared_memory_per_multiprocessor
    assert cluster == 1 or 0 <= whole - 1024 - shared < 1024


@pytest.mark.gpu
def test_streams_and_graphs():
    x = torch.randn(50, 200, device="cuda")
    b, sb = quantize_rows(torch.randn(300, 200, device="cuda"))
    want = matmul_i8(*quantize_rows(x), b, sb)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = matmul_i8(*quantize_rows(x), b, sb)
    c2, s2 = quantize_rows(x, stream=side.cuda_stream)
    got2 = matmul_i8(c2, s2, b, sb, stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(got, want) and torch.equal(got2, want)
    assert torch.equal(matmul_i8(*quantize_rows(x, stream=0), b, sb, stream=0), want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = matmul_i8(*quantize_rows(x), b, sb)
    for seed in range(3):
        x.copy_(torch.randn(50, 200, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, matmul_i8(*quantize_rows(x), b, sb))


# ------------------------------------------------------------------ refusals
def rejects(f, *a, **k):
    with pytest.raises(GustANNError) as e:
        f(*a, **k)
    assert e.value.code == api.GANN_EINVAL and str(e.value)


def test_refusals():
    x = torch.zeros(4, 32)
    c, s = torch.zeros(4, 32, dtype=torch.int8), torch.zeros(4)
    rejects(quantize_rows, x)                               # not on a GPU
    rejects(quantize_rows, x.double())
    rejects(quantize_rows, x[0])
    rejects(matmul_i8, c, s, c, s)
    rejects(matmul_i8, c.float(), s, c, s)
    rejects(matmul_i8, c, s[:3], c, s)
    rejects(matmul_i8, c, s.double(), c, s)
    rejects(matmul_i8, c, s, c[:, :16], s)
    rejects(matmul_i8, c[:, :20].contiguous(), s, c, s)     # rows of 20 bytes
    rejects(matmul_i8, c.t().contiguous().t(), s, c, s)
    rejects(matmul_i8, c, s, c, s, bias=torch.zeros(3))
    rejects(matmul_i8, c, s, c, s, bias=torch.zeros(4).half())


def test_c_entries_refuse_before_touching_the_gpu():
    lib = api.lib
    buf = (C.c_byte * 4096)()
    p = (C.addressof(buf) + 63) // 64 * 64

    def q(rows=2, xs=128, dim=32, dt=api.F32, codes=p, cs=32, x=p, scales=p):
        return lib.gann_quantize_rows(x, rows, xs, dim, dt, codes, cs, scales, 0, None)

    def mm(m=2, sa=32, n=2, sb=32, k=32, os=2, dt=api.F32, a=p, out=p, bias=None):
        return lib.gann_matmul_i8(a, m, sa, p, p, n, sb, p, bias, k, out, os, dt, 0, None)

    bad = [q(rows=-1), q(dim=0), q(dim=131072, cs=131072), q(dt=0), q(dt=4), q(cs=16), q(cs=40), q(xs=-4), q(xs=130),
           q(x=None), q(codes=None), q(scales=None), q(codes=p + 8), q(x=p + 2),
           mm(m=-1), mm(n=-1), mm(k=0), mm(k=131072, sa=131072, sb=131072), mm(sa=16), mm(sa=40), mm(sb=33), mm(os=1),
           mm(dt=0), mm(a=None), mm(a=p + 4), mm(out=None), mm(out=p + 1), mm(bias=p + 2)]
    assert bad == [api.GANN_EINVAL] * len(bad)
    assert q(rows=0) == api.GANN_OK and mm(m=0) == api.GANN_OK and mm(n=0, os=0) == api.GANN_OK


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    c, s = i8(4, 32, 1)
    rejects(matmul_i8, c.cpu(), s, c, s)
    rejects(quantize_rows, torch.zeros(32, 4, device="cuda").t())
    rejects(matmul_i8, c, s, c, s, out=torch.zeros(4, 5, device="cuda"))
    rejects(matmul_i8, c, s, c, s, out=torch.zeros(4, 4, device="cuda", dtype=torch.int32))
    rejects(matmul_i8, c, s, c, s, out=torch.zeros(4, 4, device="cuda").t())
    rejects(matmul_i8, c, s, c, s, dtype=torch.float16, out=torch.zeros(4, 4, device="cuda"))
    rejects(matmul_i8, c, s, c, s, out=torch.zeros(1, 4, device="cuda").expand(4, 4))
    both = torch.zeros(20, device="cuda")
    rejects(matmul_i8, c, both[:4], c, s, out=both[4:20].view(4, 4)[:, :4].as_strided((4, 4), (4, 1), 2))
