"""Norm, 4-bit and grouped products one behind the other, each reading what the last one wrote.

Their kernels are placed while the previous kernel of the stream still runs and wait for it before they touch memory, so
a chain without a pause has to give the bits of one that is synchronised after every call.
"""
import pytest

from minixla_b200 import lib as mlib
from tests.operator_calls import captured, current_stream, ok, ptr, steps

D = 512        # width of every product
GROUP = 64
EXPERTS = 4
TURNS = 10


class Chain:
    def __init__(self, lib, ctx, rows):
        import torch

        g = torch.Generator(device="cuda").manual_seed(rows)

        def randn(*shape):
            return torch.randn(*shape, generator=g, device="cuda")

        self.lib, self.ctx, self.rows = lib, ctx, rows
        self.q = torch.randint(0, 256, (D, D // 2), generator=g, device="cuda", dtype=torch.uint8)
        self.scales = randn(D, D // GROUP) * (0.2 / D ** 0.5)
        self.b = randn(EXPERTS, D, D) / D ** 0.5
        cuts = torch.randint(0, rows + 1, (EXPERTS - 1,), generator=g, device="cuda").sort().values
        self.offsets = torch.cat([cuts.new_zeros(1), cuts, cuts.new_full((1,), rows)]).int()
        self.start = randn(rows, D), randn(1, D)
        self.x, self.gamma = (t.clone() for t in self.start)
        self.y, self.z, self.w = (torch.empty(rows, D, device="cuda") for _ in range(3))
        self.statistics = torch.empty(2, rows, device="cuda")

    def reset(self):
        self.x.copy_(self.start[0])
        self.gamma.copy_(self.start[1])

    def run(self, after=lambda: None):
        lib, ctx, rows, st = self.lib, self.ctx, self.rows, current_stream()
        add = steps((mlib.MXB_EP_ADD_FULL, self.x, D, 1.0))
        none = steps()
        for _ in range(TURNS):
            # gamma is what the last turn's product for one row left.
            ok(lib.mxb_layer_norm(ctx, ptr(self.x), D, ptr(self.gamma), None, 1e-5, ptr(self.y), D,
                                  ptr(self.statistics[0]), ptr(self.statistics[1]), rows, D, st))
            after()
            ok(lib.mxb_q4_gemm(ctx, ptr(self.y), D, ptr(self.q), D // 2, ptr(self.scales), mlib.MXB_SCALE_F32, None,
                               D // GROUP, GROUP, ptr(self.z), D, rows, D, D, *none, st))
            after()
            ok(lib.mxb_grouped_gemm(ctx, ptr(self.z), D, ptr(self.b), D, D * D, ptr(self.offsets), EXPERTS, ptr(self.w),
                                    D, rows, D, D, *add, mlib.GPU_PRECISION_3XTF32, st))
            after()
            ok(lib.mxb_q4_gemm(ctx, ptr(self.w), D, ptr(self.q), D // 2, ptr(self.scales), mlib.MXB_SCALE_F32, None,
                               D // GROUP, GROUP, ptr(self.gamma), D, 1, D, D, *none, st))
            after()
            # The backward kernels read the norm's rows and write the next turn's.
            ok(lib.mxb_layer_norm_backward(ctx, ptr(self.w), D, ptr(self.x), D, ptr(self.gamma),
                                           ptr(self.statistics[0]), ptr(self.statistics[1]), ptr(self.x), D, None, None,
                                           rows, D, st))
            after()
        return self.x, self.gamma


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 2, 8, 16, 40, 700, 5000])
def test_chain_without_a_pause(lib, gpu_ctx, rows):
    import torch

    chain = Chain(lib, gpu_ctx, rows)
    chain.reset()
    want = [t.clone() for t in chain.run(torch.cuda.synchronize)]
    assert all(torch.isfinite(t).all() for t in want)
    for _ in range(3):
        chain.reset()
        torch.cuda.synchronize()
        got = chain.run()
        torch.cuda.synchronize()
        assert all(torch.equal(g, w) for g, w in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [2, 40, 700])
def test_captured_chain(lib, gpu_ctx, rows):
    import torch

    chain = Chain(lib, gpu_ctx, rows)
    chain.reset()
    want = [t.clone() for t in chain.run(torch.cuda.synchronize)]

    def turn():
        chain.reset()
        chain.run()

    graph = captured(turn, replays=3)
    assert all(torch.equal(g, w) for g, w in zip((chain.x, chain.gamma), want))
    del graph


@pytest.mark.gpu
def test_chain_with_cta_pairs(lib, gpu_ctx):
    """A chain whose grouped product runs on CTA pairs: without a pause, and captured."""
    import torch

    rows = 8000
    assert mlib.grouped_plan(mlib.MXB_GROUPED_FORWARD, rows, EXPERTS, D, D).kernel == mlib.MXB_KERNEL_CTA_PAIR
    chain = Chain(lib, gpu_ctx, rows)
    chain.reset()
    want = [t.clone() for t in chain.run(torch.cuda.synchronize)]
    assert all(torch.isfinite(t).all() for t in want)
    for _ in range(3):
        chain.reset()
        torch.cuda.synchronize()
        got = chain.run()
        torch.cuda.synchronize()
        assert all(torch.equal(g, w) for g, w in zip(got, want))

    def turn():
        chain.reset()
        chain.run()

    graph = captured(turn, replays=3)
    assert all(torch.equal(g, w) for g, w in zip((chain.x, chain.gamma), want))
    del graph


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 16, 300])
def test_calls_behind_another_stream(lib, gpu_ctx, rows):
    """A call whose stream waits for an event of another stream reads what that stream wrote."""
    import torch

    chain = Chain(lib, gpu_ctx, rows)
    other, here = torch.cuda.Stream(), torch.cuda.Stream()
    none = steps()
    x = torch.empty_like(chain.x)

    def product(src, out):
        ok(lib.mxb_q4_gemm(gpu_ctx, ptr(src), D, ptr(chain.q), D // 2, ptr(chain.scales), mlib.MXB_SCALE_F32, None,
                           D // GROUP, GROUP, ptr(out), D, rows, D, D, *none, current_stream()))

    def normed(src, out):
        ok(lib.mxb_layer_norm(gpu_ctx, ptr(src), D, None, None, 1e-5, ptr(out), D, None, None, rows, D, current_stream()))

    normed(chain.start[0], x)
    product(x, chain.w)
    torch.cuda.synchronize()
    want = chain.w.clone()
    for _ in range(5):
        x.zero_()
        chain.w.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(other):
            torch.cuda._sleep(2_000_000)
            normed(chain.start[0], x)
            written = other.record_event()
        with torch.cuda.stream(here):
            product(chain.start[0], chain.z)  # the kernel before, on this stream, has nothing to do with x
            here.wait_event(written)
            product(x, chain.w)
        torch.cuda.synchronize()
        assert torch.equal(chain.w, want)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 16, 300])
def test_captured_fork(lib, gpu_ctx, rows):
    """The same inside a graph: a branch on another stream writes what the call behind the join reads."""
    import torch

    chain = Chain(lib, gpu_ctx, rows)
    other = torch.cuda.Stream()
    none = steps()
    x = torch.empty_like(chain.x)

    def product(src, out):
        ok(lib.mxb_q4_gemm(gpu_ctx, ptr(src), D, ptr(chain.q), D // 2, ptr(chain.scales), mlib.MXB_SCALE_F32, None,
                           D // GROUP, GROUP, ptr(out), D, rows, D, D, *none, current_stream()))

    def normed():
        ok(lib.mxb_layer_norm(gpu_ctx, ptr(chain.x), D, None, None, 1e-5, ptr(x), D, None, None, rows, D,
                              current_stream()))

    def fork():
        here = torch.cuda.current_stream()
        other.wait_stream(here)
        with torch.cuda.stream(other):
            for _ in range(20):
                normed()
        product(chain.start[0], chain.z)
        here.wait_stream(other)
        product(x, chain.w)

    graph = captured(fork)
    for turn in range(3):
        chain.x.copy_(chain.start[0] * (turn + 1) + turn)
        graph.replay()
        torch.cuda.synchronize()
        got = chain.w.clone()
        normed()
        torch.cuda.synchronize()
        product(x, chain.w)
        torch.cuda.synchronize()
        assert torch.equal(got, chain.w)
    del graph


@pytest.mark.gpu
def test_two_threads_on_their_per_thread_streams(lib, gpu_ctx):
    """cudaStreamPerThread is one handle and another stream in each thread: the calls' pooled workspaces stay apart."""
    import threading

    import torch

    per_thread, turns, rows, cols, m = 2, 40, 2000, 1000, 64
    none = steps()

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    g = torch.Generator(device="cuda").manual_seed(0)
    x, dy, mean = randn(2, rows, cols), randn(2, rows, cols), randn(2, rows)
    rstd = torch.ones(rows, device="cuda")
    a, scales = randn(2, m, D), randn(D, D // GROUP)
    q = torch.randint(0, 256, (D, D // 2), generator=g, device="cuda", dtype=torch.uint8)

    def calls(i, dgamma, dbeta, out, stream):
        ok(lib.mxb_layer_norm_backward(gpu_ctx, ptr(dy[i]), cols, ptr(x[i]), cols, None, ptr(mean[i]), ptr(rstd), None, 0,
                                       ptr(dgamma), ptr(dbeta), rows, cols, stream))
        ok(lib.mxb_q4_gemm(gpu_ctx, ptr(a[i]), D, ptr(q), D // 2, ptr(scales), mlib.MXB_SCALE_F32, None, D // GROUP, GROUP,
                           ptr(out), D, m, D, D, *none, stream))

    def outputs(n):
        return [(torch.zeros(cols, device="cuda"), torch.zeros(cols, device="cuda"), torch.zeros(m, D, device="cuda"))
                for _ in range(n)]

    want, got = outputs(2), [outputs(turns) for _ in range(2)]
    for i in range(2):
        calls(i, *want[i], current_stream())
        torch.cuda.synchronize()
    errors, begin = [], threading.Barrier(2)

    def work(i):
        try:
            torch.cuda.set_device(0)
            begin.wait()
            for o in got[i]:
                calls(i, *o, per_thread)
            torch.cuda.synchronize()
        except BaseException as e:  # noqa: BLE001 - reported by the main thread
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for i in range(2):
        for turn, o in enumerate(got[i]):
            assert all(torch.equal(v, w) for v, w in zip(o, want[i])), (i, turn)
    assert lib.mxb_check_device_error(gpu_ctx) == 0


@pytest.mark.gpu
def test_a_failed_call_leaves_no_error_behind(lib, gpu_ctx):
    """A call on the legacy stream while a blocking stream is being captured is an error of that call alone."""
    import ctypes as C

    import torch

    driver = C.CDLL("libcuda.so.1")
    x, gamma = torch.randn(40, D, device="cuda"), torch.ones(D, device="cuda")
    dy, mean, rstd, grads = torch.randn_like(x), torch.zeros(40, device="cuda"), torch.ones(40, device="cuda"), torch.zeros(2, D, device="cuda")

    def backward(stream):
        return lib.mxb_layer_norm_backward(gpu_ctx, ptr(dy), D, ptr(x), D, ptr(gamma), ptr(mean), ptr(rstd), None, 0,
                                           ptr(grads[0]), ptr(grads[1]), 40, D, stream)

    ok(backward(mlib.CUDA_STREAM_LEGACY))
    torch.cuda.synchronize()
    want = grads.clone()
    grads.zero_()
    torch.cuda.synchronize()
    stream, graph = C.c_void_p(), C.c_void_p()
    assert driver.cuStreamCreate(C.byref(stream), 0) == 0
    assert driver.cuStreamBeginCapture_v2(stream, 0) == 0
    try:
        assert backward(mlib.CUDA_STREAM_LEGACY) < 0 and "captur" in mlib.last_error()
    finally:
        if driver.cuStreamEndCapture(stream, C.byref(graph)) == 0 and graph:
            driver.cuGraphDestroy(graph)
        assert driver.cuStreamDestroy_v2(stream) == 0
    ok(backward(mlib.CUDA_STREAM_LEGACY))
    torch.cuda.synchronize()
    assert torch.equal(grads, want)
