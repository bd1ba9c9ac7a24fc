"""Where the logit losses put a gradient, on the meta device: no memory is taken."""

from __future__ import annotations

import torch

from picotron_b200 import ops


def test_gradients_of_slices_take_little_more_than_their_own_memory():
    """Odd rows need the logits' addresses modulo 16 bytes, not the span of the view."""

    size = {torch.float32: 4, torch.bfloat16: 2, torch.float16: 2}
    whole = (8, 4096, 50257)
    views = {
        "last": lambda x: x[:, -1:], "first": lambda x: x[:, :1], "few": lambda x: x[:, -5:],
        "every 512th": lambda x: x[:, ::512], "without the last": lambda x: x[:, :-1],
        "one sequence": lambda x: x[3], "one of each": lambda x: x[:, 7],
        "other order": lambda x: x[:, -3:].transpose(0, 1), "classes": lambda x: x[:, :3, 1:9],
        "no positions": lambda x: x[:, :0], "every other sequence": lambda x: x[::2, :40],
    }
    for dtype, width in size.items():
        x = torch.empty(whole, dtype=dtype, device="meta")
        for name, view in views.items():
            v = view(x)
            d = ops._ll_gradient(v)
            assert d.shape == v.shape and d.dtype == dtype and d.stride(-1) == 1, name
            held = d.untyped_storage().nbytes()
            assert held <= 2 * v.numel() * width + 16 * (v.numel() // max(1, v.size(-1)) + 1), name
            # Rows at the logits' places modulo 16 bytes, none over another.
            per = 16 // width
            rows = sorted((d.stride(i), v.stride(i), v.size(i)) for i in range(v.dim() - 1)
                          if v.size(i) > 1)
            assert v.numel() == 0 or (d.storage_offset() - v.storage_offset()) % per == 0, name
            reach = v.size(-1)
            for ds, vs, n in rows if v.numel() else ():
                assert (ds - vs) % per == 0 and ds >= reach, name
                reach += ds * (n - 1)
            fake = ops._logit_loss_backward_fake(v, None, None, None, None, None)
            assert fake.stride() == d.stride() or v.numel() == 0, name
