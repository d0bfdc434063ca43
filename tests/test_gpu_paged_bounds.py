"""Calls of the paged cache whose batch is against its contract: only the batch's own memory is
touched."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_steps_past_the_most(mga, dev):
    """32 overlapping sequences of so many steps that their list ends before the last tiles, in a workspace that
    holds what would lead far out of it: the rows of ``out`` alone are written."""
    B, T, D, ps, W = 64, 8192, 64, 128, 65700
    len_ = (W - 64) * ps
    table = torch.full((B, W), -1, dtype=torch.int32, device=dev)
    cu = torch.tensor([0] + [T, 0] * (B // 2), dtype=torch.int32, device=dev)
    lengths = torch.full((B,), len_, dtype=torch.int32, device=dev)
    # tiles of 32 rows: the call's are few enough to be taken, the overlapping ones are not
    steps = (len_ + T + 63) // 64
    assert (T // 32 + B) * ((W * ps + T) // 64 + 2) <= 1 << 30 < B // 2 * (T // 32) * (steps - T // 64)
    kv = torch.zeros(ps * D, dtype=torch.uint8, device=dev)
    scale = torch.ones(1, device=dev)
    q = torch.randn(T, D, device=dev).bfloat16()
    out = torch.full((3, T, D), 7.0, dtype=torch.bfloat16, device=dev)
    lib = mga._lib
    n = int(lib.load().mga_paged_attn_workspace_bytes(T, B, 1, 1, D, ps, W, 0))
    assert n > 0
    ws = torch.full((n + 4096,), 0x7f, dtype=torch.uint8, device=dev)
    print("overlapping sequences, notes of 0x7f7f7f7f", flush=True)
    lib.call("mga_paged_attn", q.data_ptr(), D, D, kv.data_ptr(), kv.data_ptr(), scale.data_ptr(), scale.data_ptr(), 1, ps,
             table.data_ptr(), W, W, cu.data_ptr(), lengths.data_ptr(), T, B, 1, 1, D, 0, 0.125, out[1].data_ptr(), D, D, 0,
             ws.data_ptr(), n, torch.cuda.current_stream(dev).cuda_stream)
    torch.cuda.synchronize()
    assert (out[::2] == 7).all() and (ws[n:] == 0x7f).all()
