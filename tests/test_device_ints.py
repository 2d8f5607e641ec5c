"""Device slot ids, offsets and orders are read as packed int32: other tensors are refused."""

import pytest
import torch

from wkvm_amd import linear_decode_slots, linear_prefill_varlen, ops

I32, BF16 = torch.int32, torch.bfloat16
CPU = torch.device("cpu")


def test_packed_ints():
    ok = torch.arange(3, dtype=I32)
    assert ops.packed_ints(ok, 3, CPU, "x") is ok
    assert ops.packed_ints(ok[1:2], 1, CPU, "x").tolist() == [1]
    many = torch.arange(6, dtype=I32)
    for wrong in (many[::2], many[:1].expand(3), ok[:2], many, ok.long(), ok.float(), [0, 1, 2],
                  many.view(3, 2)[:, 0], ok.view(3, 1), ok.to("meta")):
        with pytest.raises(ValueError, match="x must be a contiguous device int32 tensor of 3"):
            ops.packed_ints(wrong, 3, CPU, "x")


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["ids", "order", "cu"])
def test_strided_integers_are_refused(dev, which):
    """Every entry point that takes device integers, with every second entry of a larger tensor."""
    T, n = 8, 2
    pool = torch.randn(5, 2, 64, 64, device=dev)
    before = pool.clone()
    x = torch.randn(T, 2, 64, device=dev).to(BF16)
    g = torch.zeros(2, device=dev)
    rows = torch.zeros(5, 128, dtype=BF16, device=dev)
    mix = torch.zeros(1, 128, dtype=BF16, device=dev)

    def ints(values, name):
        t = torch.tensor(values, dtype=I32, device=dev)
        return t.repeat_interleave(2)[::2] if which == name else t

    ids, order, cu = ints([1, 2], "ids"), ints([1, 0], "order"), ints([0, 3, T], "cu")
    six, row = (x,) * 6, (x[:n],) * 6
    calls = {
        "decode": lambda: ops.wkv7_decode_slots(pool, ids, *row, row_order=order),
        "decode_into": lambda: ops.wkv7_decode_into(pool, None, *row, in_ids=ids, row_order=order),
        "decode_layers": lambda: ops.wkv7_decode_layers(pool[None], ids, [row], row_order=order),
        "linear_decode": lambda: linear_decode_slots(pool, ids, *row[:3], g, row_order=order),
        "prefill": lambda: ops.wkv7_prefill_varlen(pool, ids, cu, *six, seq_order=order),
        "prefill_into": lambda: ops.wkv7_prefill_into(pool, None, cu, *six, in_ids=ids,
                                                      seq_order=order),
        "linear_prefill": lambda: linear_prefill_varlen(pool, ids, cu, x, x, x, g,
                                                        seq_order=order),
        "token_shift": lambda: ops.token_shift_mix(x.view(T, 128), rows, ids, mix, cu),
        "slot_zero": lambda: ops.slot_zero(pool, ids, 0),
        "slot_copy": lambda: ops.slot_copy(pool, None, torch.zeros_like(pool), ids, 0),
    }
    takes = {"order": [c for c in calls if c[:5] not in ("token", "slot_")],
             "cu": ["prefill", "prefill_into", "linear_prefill", "token_shift"], "ids": list(calls)}
    for name in takes[which]:
        with pytest.raises(ValueError, match="contiguous"):
            calls[name]()
    torch.cuda.synchronize()
    assert torch.equal(pool, before)
