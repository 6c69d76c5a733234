"""What an orthogonalised update does where the blocks that an epilogue asks for never come: each warp reports it once and touches nothing more."""
import ctypes as C
import time

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", [(1, 300, 520), (1, 1400, 1300), (1, 200, 6000), (12, 700, 301)])
def test_blocks_that_never_come(built_lib, diag_lib, shape):
    """The diagnostics build sends for none of them, with a poll budget of about two milliseconds a wait: some launch has several tiles a CTA, none more than its own two waits."""
    g = torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(sum(shape)), device="cuda")
    st, numbers = torch.cuda.current_stream().cuda_stream, (C.c_float * 6)(*((3.4445, -4.7750, 2.0315) * 2))
    size = diag_lib.pb_orthogonalize_workspace_size(*shape)
    ws = torch.zeros(size, dtype=torch.uint8, device="cuda")

    def run():
        out = torch.zeros(shape, dtype=torch.bfloat16, device="cuda")
        assert diag_lib.pb_orthogonalize(g.data_ptr(), 0, *shape, 2, C.addressof(numbers), 1e-7, out.data_ptr(), ws.data_ptr(), size, st) == 0
        torch.cuda.synchronize()
        return out

    before = run()
    assert diag_lib.pb_gemm_check(st) == 0
    try:
        assert diag_lib.pb_debug_product_control(1 << 10, 4) == 0
        start = time.monotonic()
        got = run()
        took = time.monotonic() - start
        assert diag_lib.pb_gemm_check(st) == 7 and b"orthogonalised" in diag_lib.pb_last_error()
        assert diag_lib.pb_gemm_check(st) == 0
    finally:
        diag_lib.pb_debug_product_control(0, 0)
    assert not got.any()                                          # the last product's epilogue writes nothing that it could not add to
    assert took < 5.0                                             # four launches with two waits of milliseconds; a wait a block would be hundreds
    assert torch.equal(before, run()) and diag_lib.pb_gemm_check(st) == 0
