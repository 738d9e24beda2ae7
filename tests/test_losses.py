"""Argument checks of the losses that need no GPU."""
import pytest
import torch

import gefen


def test_host_logits_are_refused():
    logits, labels = torch.zeros(2, 3, 5), torch.zeros(2, 3, dtype=torch.long)
    with pytest.raises(ValueError, match="HIP device"):
        gefen.token_logps(logits, labels)
    with pytest.raises(ValueError, match="HIP device"):
        gefen.preference_loss(logits, labels)
    with pytest.raises(ValueError, match="HIP device"):
        gefen.policy_loss_and_grad(logits, labels, torch.zeros(2, 3), torch.zeros(2))


def test_other_things_than_tensors_are_refused():
    with pytest.raises(TypeError):
        gefen.token_logps([[1.0]], torch.zeros(1, dtype=torch.long))


def test_bad_descriptors_are_refused_on_the_host():
    import ctypes
    from gefen.kernels import _native
    lib = _native.load()
    good = dict(logits=64, labels=64, rows=4, rows_per_batch=2, batch_stride=10, row_stride=5, vocab=5, dtype=0, n_seq=2)
    assert lib.gefenx_loss_workspace_bytes(ctypes.byref(_native.Logits(**good))) > 0
    for change in ({"dtype": 3}, {"vocab": 0}, {"rows": -1}, {"rows_per_batch": 0}, {"labels": None}, {"rows": 1 << 31}, {"rows": 1 << 30}, {"n_seq": -1}, {"n_seq": 1 << 30}):
        d = _native.Logits(**{**good, **change})
        assert lib.gefenx_loss_workspace_bytes(ctypes.byref(d)) == 0, change
        assert lib.gefenx_token_logps(ctypes.byref(d), 64, 64, 64, 1 << 20, None) == (-2 if "dtype" in change else -1), change
    odd = _native.Logits(**{**good, "rows": 6, "n_seq": 3})
    assert lib.gefenx_preference_loss(ctypes.byref(odd), None, 0.1, 0.0, 0, 64, 64, 64, 64, 64, 64, 64, 1 << 20, None) == -1
    none = _native.Logits(**{**good, "n_seq": 0})
    assert lib.gefenx_preference_loss(ctypes.byref(none), None, 0.1, 0.0, 0, 64, 64, 64, 64, 64, 64, 64, 1 << 20, None) == -1
    small = _native.Logits(**good)
    assert lib.gefenx_token_logps(ctypes.byref(small), 64, 64, 64, 8, None) == -1
    assert "workspace" in _native.last_error()


@pytest.mark.parametrize("change", ["strides", "batches", "vocabulary", "type", "label strides", "label type", "offset type", "offset count"])
def test_backward_takes_no_descriptor_by_its_address_alone(change, monkeypatch):
    """Saved tensors that came back at the addresses of the forward pass's, but laid out otherwise, are described anew
    (which host tensors refuse); the same ones are not."""
    import types
    from gefen import losses
    from gefen.kernels import _native
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: types.SimpleNamespace(cuda_stream=0))
    memory, labels, cu = torch.zeros(4096), torch.zeros(64, dtype=torch.int64), torch.tensor([0, 3, 6], dtype=torch.int32)
    packed = change.startswith("offset")
    x, y = (memory.as_strided((6, 8), (12, 1)), labels[:6]) if packed else (memory.as_strided((2, 3, 8), (48, 12, 1)),
                                                                          labels[:6].view(2, 3))
    desc = _native.Logits(x.data_ptr(), y.data_ptr(), cu.data_ptr() if packed else None, 6, 6 if packed else 3,
                          0 if packed else 48, 12, 8, -100, _native.DT_F32, 2)
    offsets = cu if packed else None
    assert losses._Call.again(desc, x, y, -100, offsets).desc is desc
    if change == "strides":
        x = memory.as_strided((2, 3, 8), (24, 8, 1))
    elif change == "batches":  # [:, :-1] of four rows, come back without the fourth
        x = memory.as_strided((2, 3, 8), (36, 12, 1))
    elif change == "vocabulary":
        x = memory.as_strided((2, 3, 7), (48, 12, 1))
    elif change == "type":
        x = memory.view(torch.bfloat16).as_strided((2, 3, 8), (48, 12, 1))
    elif change == "label strides":
        y = labels.as_strided((2, 3), (6, 2))
    elif change == "label type":
        y = labels.view(torch.int32)[:6].view(2, 3)
    elif change == "offset type":
        offsets = torch.tensor([0, 3, 6])
        desc.cu_seqlens = offsets.data_ptr()
    else:
        offsets = torch.zeros(4, dtype=torch.int32)
        desc.cu_seqlens = offsets.data_ptr()
    with pytest.raises(ValueError, match="HIP device"):
        losses._Call.again(desc, x, y, -100, offsets)
