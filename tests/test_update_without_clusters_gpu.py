"""Orthogonalised updates where a cluster of sixteen CTAs does not fit, as on a part of a GPU: the diagnostics build takes eight for the most."""
import ctypes as C

import pytest
import torch

pytestmark = pytest.mark.gpu

TRIPLES = (3.4445, -4.7750, 2.0315) * 5


def _run(lib, g):
    batch, rows, cols = g.shape
    numbers, st = (C.c_float * 15)(*TRIPLES), torch.cuda.current_stream().cuda_stream
    size = lib.pb_orthogonalize_workspace_size(batch, rows, cols)
    out, ws = torch.zeros(g.shape, dtype=torch.bfloat16, device="cuda"), torch.zeros(size, dtype=torch.uint8, device="cuda")
    assert lib.pb_orthogonalize(g.data_ptr(), 0 if g.dtype is torch.float32 else 1, batch, rows, cols, 5, C.addressof(numbers), 1e-7, out.data_ptr(), ws.data_ptr(), size, st) == 0
    assert lib.pb_gemm_check(st) == 0
    return out, size


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape,sixteen", [((1, 2048, 128), False), ((2, 100, 1500), False), ((1, 2049, 128), True), ((2, 4096, 128), True), ((1, 70, 3001), True)])
def test_without_clusters_of_sixteen(built_lib, diag_lib, shape, sixteen, dtype):
    """What needs one goes through the products, with their errors (2-norms: test_orthogonalize_gpu.py derives 5e-3); the rest has the same bits."""
    g = torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(sum(shape)), device="cuda").to(dtype)
    want, _ = _run(diag_lib, g)
    assert torch.equal(want, _run(built_lib, g)[0])
    try:
        assert diag_lib.pb_debug_product_control(0, 2) == 0
        got, size = _run(diag_lib, g)
    finally:
        diag_lib.pb_debug_product_control(0, 0)
    assert (size > 256) == sixteen
    if not sixteen:
        assert torch.equal(got, want)
    x = g.double() / g.double().norm(dim=(1, 2), keepdim=True)
    x = x.mT if x.shape[1] > x.shape[2] else x
    for _ in range(5):
        p = x @ x.mT
        x = TRIPLES[0] * x + (TRIPLES[1] * p + TRIPLES[2] * p @ p) @ x
    x = x.mT if x.shape[1:] != g.shape[1:] else x
    assert ((got.double() - x).norm(dim=(1, 2)) <= 5e-3 * x.norm(dim=(1, 2))).all()
