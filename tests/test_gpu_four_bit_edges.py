"""The 4-bit operators where streams, forms of a launch and scales meet their limits."""
import numpy as np
import pytest
import torch

from ember_amd import kernels as K
from four_bit_reference import D
from test_gpu_four_bit import batch, check, dint, on

pytestmark = pytest.mark.gpu


def keep_busy():
    """Some 20 ms or more of work on the current stream."""
    x = torch.ones(4096, 4096, device="cuda")
    for _ in range(20):
        x = x @ x * 2.0 ** -12
    return x


@pytest.mark.parametrize("handle", [False, True], ids=["object", "handle"])
def test_a_workspace_is_zeroed_in_the_order_of_its_calls_stream(rng, device, handle):
    """The current stream is busy, and the memory that the workspace gets held other bytes: calls on another stream find
    zeros all the same, and all rows of items that are shared out are written."""
    b = batch(rng, device, [(9000, 1), (7000, 1)], 4, 2)
    out = torch.full((2, 4, D), 7.0, dtype=torch.float16, device=device)
    args = (on(b["q"], device), on(b["pages"], device), out, dint(b["start"], device), dint(b["pos"], device), dint(b["table"], device))
    sizes = dict(max_query=1, max_context=b["longest"])
    s = torch.cuda.Stream()
    n = K.kv4_workspace(2, 2, n_heads=4, n_kv=2, device=device, **sizes).numel()
    with torch.cuda.stream(s):
        torch.full((n,), 255, dtype=torch.uint8, device=device)
    torch.cuda.synchronize()
    busy = keep_busy()
    stream = s.cuda_stream if handle else s
    ws = K.kv4_workspace(2, 2, n_heads=4, n_kv=2, device=device, **sizes, stream=stream)
    assert ws.numel() == n
    for _ in range(3):
        K.kv4_attention(*args, **sizes, workspace=ws, stream=stream)
    s.synchronize()
    check(b, out.double().cpu().numpy())
    torch.cuda.synchronize()
    del busy


def test_prepared_tensors_are_not_ones_that_the_current_stream_still_writes(rng, device):
    """Blocks that the current stream has freed, with writes to them still queued there, are not what mx_quantize and
    gemv4_pack return on another stream."""
    x = on(rng.standard_normal((4096, 4096)).astype(np.float32), device)
    codes, scales = K.mx_quantize(x)
    packed = K.gemv4_pack(codes, scales)
    s = torch.cuda.Stream()
    for like, call in ((codes, lambda: K.mx_quantize(x, stream=s)[0]), (scales, lambda: K.mx_quantize(x, stream=s)[1]),
                       (packed, lambda: K.gemv4_pack(codes, scales, stream=s))):
        torch.cuda.synchronize()
        busy = keep_busy()
        freed = torch.empty_like(like)
        at = freed.data_ptr()
        freed.fill_(99)  # runs behind the products
        del freed
        assert torch.empty_like(like).data_ptr() == at  # what an allocation on the current stream would get
        got = call()
        torch.cuda.synchronize()
        assert torch.equal(got, like)
        del busy
