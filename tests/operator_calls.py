"""Helpers of the operator tests: calls through the C ABI on torch tensors."""
import ctypes as C

from minixla_b200 import lib as mlib

U = 2.0 ** -24  # half a step of fp32, relative


def ptr(t):
    return t.data_ptr() if t is not None else None


def steps(*items):
    """(kind, operand tensor or None, ld_or_size, scale) -> (array, count)."""
    arr = (mlib.EpStepDev * max(1, len(items)))()
    for i, (kind, operand, ld, scale) in enumerate(items):
        arr[i].kind, arr[i].operand, arr[i].ld_or_size, arr[i].scale = kind, ptr(operand), ld, scale
    return arr, len(items)


def current_stream():
    import torch

    return torch.cuda.current_stream().cuda_stream or mlib.CUDA_STREAM_LEGACY


def ok(rc):
    assert rc == 0, mlib.last_error()


def fake_context():
    """A non-NULL context for calls that must be refused before it is touched."""
    return C.cast(C.create_string_buffer(1 << 14), C.c_void_p)


def pitched(t, pitch, fill=float("nan")):
    """`t` ([..., cols]) as a view of a buffer with row pitch `pitch`; the gap holds `fill`."""
    import torch

    buf = torch.full((*t.shape[:-1], pitch), fill, dtype=t.dtype, device=t.device)
    buf[..., : t.shape[-1]] = t
    return buf[..., : t.shape[-1]]


def within(got, want, tol, what=""):
    """Every element of got within tol (a tensor or number) of want, both compared in float64."""
    import torch

    got = got.double()
    assert not torch.isnan(got).any(), f"{what}: NaN"
    over = ((got - want).abs() - tol).max().item()
    assert over <= 0, f"{what}: off by {over:.3g} more than the bound"


def captured(call, replays=2):
    """Captures call() (which launches on the current stream) and replays it."""
    import torch

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call()  # modules loaded, attributes set
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        call()
    for _ in range(replays):
        graph.replay()
    torch.cuda.synchronize()
    return graph
