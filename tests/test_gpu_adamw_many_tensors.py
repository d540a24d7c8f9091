"""AdamW over more chunks than one launch takes workgroups: a HIP grid has fewer than 2^32 threads, 2^22 chunks of the 8-bit form."""
import ctypes

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
COUNT = 2 ** 22 + 5


@pytest.mark.parametrize("zero_grads", [0, 1])
def test_four_million_tensors_of_one_element(zero_grads):
    import torch
    from em_adapt_tensorflow_amd import _lib, ops
    assert torch.cuda.is_available()
    lib = _lib.load()
    w = torch.ones(COUNT, device="cuda")
    g = torch.full((COUNT,), 0.5, device="cuda")
    g[COUNT // 2:] = -0.5
    codes = torch.zeros((2, COUNT, 64), dtype=torch.uint8, device="cuda")
    powers = torch.zeros((COUNT, 2), dtype=torch.uint8, device="cuda")
    k = np.arange(COUNT, dtype=np.uint64)
    arr = np.zeros(COUNT, np.dtype([("w", "<u8"), ("g", "<u8"), ("m", "<u8"), ("v", "<u8"), ("e", "<u8"), ("n", "<i8"), ("unit", "<i8"), ("wd", "<f4"), ("ls", "<f4")]))
    assert arr.itemsize == ctypes.sizeof(_lib.AdamwTensor)
    arr["w"], arr["g"], arr["e"] = w.data_ptr() + 4 * k, g.data_ptr() + 4 * k, powers.data_ptr() + 2 * k
    arr["m"], arr["v"] = codes[0].data_ptr() + 64 * k, codes[1].data_ptr() + 64 * k
    arr["n"], arr["unit"], arr["ls"] = 1, 64 * k, 1.0
    tensors = ctypes.cast(arr.ctypes.data, ctypes.POINTER(_lib.AdamwTensor))
    assert lib.emadapt_adamw_chunks(COUNT, tensors) == COUNT
    table = np.zeros(lib.emadapt_adamw_table_bytes(COUNT), np.uint8)
    assert lib.emadapt_adamw_table(COUNT, tensors, 0, 1, table.ctypes.data, table.size) == 0
    table = torch.from_numpy(table).cuda()
    control = torch.zeros(lib.emadapt_adamw_control_bytes(), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    print("step", flush=True)
    rc = lib.emadapt_adamw_step(table.data_ptr(), COUNT, 0, 1, control.data_ptr(), control.numel(), 0.25, 0.9, 0.999, 1e-8, 1.0, 0.0, 3, zero_grads,
                                torch.cuda.current_stream().cuda_stream)
    assert rc == 0 and int(control[:8].view(torch.int64)) == 1
    # from zero moments the step is lr times the gradient's sign, to the rounding of a quotient next to 1 and of eps
    want = 1.0 - 0.25 * torch.sign(torch.cat([torch.ones(COUNT // 2), -torch.ones(COUNT - COUNT // 2)])).cuda()
    assert bool(((w - want).abs() < 1e-6).all())
    assert bool((codes[:, :, 0] != 0).all()) and not bool(codes[:, :, 1:].any())
    assert bool((g == 0).all()) if zero_grads else bool((g.abs() == 0.5).all())
    assert ops.status_poll(raise_on_error=False) == 0
