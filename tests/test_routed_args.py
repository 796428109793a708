"""Refusals of the routed linears, on the CPU: every argument is checked before
any device work, so no GPU is needed."""
import ctypes
import subprocess

import pytest

from conftest import PACKAGE

P = 4096  # a 16-byte aligned address that no refused call touches


@pytest.fixture(scope="module")
def samq():
    lib = PACKAGE / "libsamq.so"
    if not lib.exists():
        subprocess.run(["make", "-C", str(PACKAGE), "-s", "-j4"], check=True)
    import samq as module
    module.library()
    return module


def refused(samq, name, args, word):
    lib = samq.library()
    assert getattr(lib, name)(*args) == 1, (name, args)
    assert word.encode() in lib.samq_last_error_v1(), lib.samq_last_error_v1()


def changed(args, **kw):
    out = dict(args)
    out.update(kw)
    return list(out.values())


ROUTE = {"logits": P, "tokens": 8, "experts": 16, "ld": 16, "top_k": 2, "normalize": 1, "weights": P, "ids": P,
         "offsets": P, "rows": P, "slots": P, "workspace": None, "bytes": 0, "stream": None}


@pytest.mark.parametrize("kw,word", [
    ({"tokens": -1}, "token count"), ({"tokens": (1 << 20) + 1}, "token count"), ({"experts": 0}, "expert count"),
    ({"experts": 1025, "ld": 1025}, "expert count"), ({"top_k": 0}, "top_k"), ({"top_k": 17}, "top_k"),
    ({"experts": 64, "ld": 64, "top_k": 33}, "top_k"), ({"ld": 15}, "stride"), ({"logits": None}, "null"),
    ({"weights": None}, "null"), ({"ids": P + 2}, "misaligned"), ({"rows": None}, "null"), ({"slots": None}, "null"),
    ({"offsets": None}, "offsets"), ({"tokens": 4096}, "workspace"), ({"tokens": 4096, "bytes": 1 << 24}, "workspace"),
    ({"tokens": 4096, "bytes": 1 << 24, "workspace": P + 8}, "aligned")])
def test_route_refusals(samq, kw, word):
    refused(samq, "samq_route_v1", changed(ROUTE, **kw), word)


COMBINE = {"y": P, "y_type": 1, "y_rows": 16, "ldy": 64, "slots": P, "weights": P, "tokens": 8, "top_k": 2,
           "width": 64, "residual": None, "ldr": 0, "out": P, "ldo": 64, "stream": None}


@pytest.mark.parametrize("kw,word", [
    ({"y_type": 30}, "y_type"), ({"tokens": -1}, "row count"), ({"y_rows": -1}, "row count"), ({"top_k": 0}, "top_k"),
    ({"top_k": 33}, "top_k"), ({"width": 0}, "width"), ({"width": 60}, "width"), ({"y_type": 0, "width": 62}, "width"),
    ({"slots": None}, "slots"), ({"weights": P + 1}, "slots"), ({"y": P + 8}, "16-byte"), ({"y": None}, "16-byte"),
    ({"ldy": 60}, "stride"), ({"ldy": 68}, "stride"), ({"out": None}, "out"), ({"ldo": 66}, "out"),
    ({"residual": P + 4, "ldr": 64}, "residual"), ({"residual": P, "ldr": 32}, "residual")])
def test_combine_refusals(samq, kw, word):
    refused(samq, "samq_combine_v1", changed(COMBINE, **kw), word)


def test_linears_refuse_null_handles(samq):
    refused(samq, "samq_linear_grouped_v1", [None, 1, P, 1, 8, 64, None, P, 8, None, 0, P, 1, 64, None, 0, None],
            "null weights")
    refused(samq, "samq_linear_adapters_v1", [None, None, P, 1, 8, 64, P, None, 0, P, 1, 64, None, 0, None],
            "null weights")
    refused(samq, "samq_adapters_set_v1", [None, 0, 0, None, None, 1, 1.0, None], "null adapters")
    lib = samq.library()
    assert lib.samq_linear_grouped_workspace_v1(None, 1, 8, 8, 0, 1) == 0
    assert lib.samq_linear_adapters_workspace_v1(None, None, 8, 0) == 0
    assert lib.samq_adapters_destroy_v1(None) == 0


@pytest.mark.parametrize("k,n,rank,count,word", [
    (0, 8, 4, 1, "width"), (48, 8, 4, 1, "width"), (64, 0, 4, 1, "row count"), (64, 8, 0, 1, "max_rank"),
    (64, 8, 129, 1, "max_rank"), (64, 8, 4, 0, "slot count"), (64, 8, 4, 4097, "slot count"),
    (64, 1 << 24, 4, 4096, "too large")])
def test_adapter_set_refusals(samq, k, n, rank, count, word):
    handle = ctypes.c_void_p()
    refused(samq, "samq_adapters_create_v1", [0, k, n, rank, count, None, ctypes.byref(handle)], word)
    assert handle.value is None
    refused(samq, "samq_adapters_create_v1", [0, 64, 8, 4, 1, None, None], "null output")


def test_route_workspace_sizes(samq):
    assert samq.route_workspace(1, 64, 2) == 0 and samq.route_workspace(64, 1024, 32) == 0
    assert samq.route_workspace(-1, 8, 1) == 0 and samq.route_workspace(8, 0, 1) == 0
    assert samq.route_workspace(16384, 128, 8) % 4 == 0 and samq.route_workspace(16384, 128, 8) > 0


def test_binding_refuses_other_tensors(samq):
    """The binding takes f16 / f32 device tensors and int32 indices only."""
    torch = pytest.importorskip("torch")
    with pytest.raises(ValueError, match="tensor on cpu"):
        samq.combine(torch.zeros(4, 8), 4, 8, torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, 2), 2, 2, 8,
                     torch.zeros(2, 8), 8)
    with pytest.raises(TypeError, match="int32"):
        samq._int32(torch.zeros(2, dtype=torch.int64))
    with pytest.raises(TypeError, match="float16 or float32"):
        samq._element(torch.bfloat16)
    assert samq._element(torch.float16) == samq.F16 and samq._element(torch.float32) == samq.F32
    assert samq._element(samq.F32) == samq.F32


ROUTE_SIZE_OF_REFUSED = """
import sys
sys.path.insert(0, {path!r})
import samq
for tokens, experts, top_k in [(100, 64, 50000), (1 << 20, 64, 1 << 30), (100, 8, 9), (100, 64, 33), (100, 1025, 2),
                               ((1 << 20) + 1, 64, 2), (1 << 62, 64, 2), (100, 1 << 30, 32)]:
    assert samq.route_workspace(tokens, experts, top_k) == 0, (tokens, experts, top_k)
print("zero")
"""


def test_route_workspace_of_refused_arguments():
    """Arguments samq_route_v1 refuses need no workspace; the question ends in no division by zero (in a process of its
    own, which one would end)."""
    import sys
    run = subprocess.run([sys.executable, "-c", ROUTE_SIZE_OF_REFUSED.format(path=str(PACKAGE))], capture_output=True,
                         text=True, timeout=240)
    assert run.returncode == 0 and "zero" in run.stdout, (run.returncode, run.stderr[-2000:])


def test_binding_refuses_tensors_that_hold_too_little(samq):
    """The checks behind the routed calls, on CPU tensors (device index -1)."""
    torch = pytest.importorskip("torch")
    samq._load_torch()
    ids = torch.zeros(8, 4, dtype=torch.int32)
    samq._array(-1, torch.int32, 32, ids, ids.view(-1), None)
    samq._array(-1, torch.int32, 0, ids[:0])
    for bad in (ids.t(), ids[:, :2], ids[:7], ids[0].expand(8, 4)):
        with pytest.raises(ValueError, match="contiguous tensor of 32 elements"):
            samq._array(-1, torch.int32, 32, bad)
    with pytest.raises(TypeError, match="int32"):
        samq._array(-1, torch.int32, 32, ids.long())
    with pytest.raises(TypeError, match="float32"):
        samq._array(-1, torch.float32, 32, ids)
    with pytest.raises(ValueError, match="tensor on cpu, expected cuda:0"):
        samq._array(0, torch.int32, 32, ids)

    x = torch.zeros(10, 24)
    for ok, rows, ld, width in ((x, 10, 24, 24), (x, 9, 24, 8), (x[:, 8:], 10, 24, 16), (x[2:, :8], 8, 24, 8),
                                (x.view(-1), 20, 12, 12), (x[0], 1, 99, 24), (x, 0, 24, 24),
                                (x[9:, 23:], 1, 8, 1), (x.view(2, 5, 24)[:, :, :8], 10, 24, 8), (x[:0], 0, 24, 24)):
        samq._rows(-1, ok, rows, ld, width)
    for bad, rows, ld, width in ((x, 11, 24, 24), (x[:, 8:], 10, 24, 17), (x[:, 20:], 10, 24, 8), (x[1:], 10, 24, 24),
                                 (x.t(), 10, 24, 24), (x[:, :8], 10, 8, 8), (x[0].expand(10, 24), 10, 24, 24),
                                 (x, 1 << 40, 24, 24), (x[:0], 1, 24, 24), (x, 10, 32, 24), (x[:7], 10, 24, 24),
                                 (x[:, 20:], 10, 24, 5)):
        with pytest.raises(ValueError, match="rows of"):
            samq._rows(-1, bad, rows, ld, width)
    with pytest.raises(TypeError, match="float32"):
        samq._float32_rows(-1, x.half(), 10, 24, 24)


def test_combine_in_place_takes_one_stride(samq):
    """The residual in place of the sum: of another row stride, rows would be written before others have read them."""
    refused(samq, "samq_combine_v1", changed(COMBINE, residual=P, out=P, ldr=64, ldo=128), "residual")
    refused(samq, "samq_combine_v1", changed(COMBINE, residual=P, out=P, ldr=128, ldo=64), "residual")
