"""Checks and the device guard that the model-side operators share."""
import contextlib

import torch

_NONE = contextlib.nullcontext()


def on_device_of(t):
    """Makes the tensor's device (and with it torch's current stream there) the current one for a call."""
    return _NONE if t.device.index == torch.cuda.current_device() else torch.cuda.device(t.device)


def check_out(out, shape, dtype, device):
    if not (out.device == device and out.dtype == dtype and tuple(out.shape) == tuple(shape) and out.is_contiguous()):
        raise ValueError("out must be a contiguous %s tensor %s on %s" % (dtype, tuple(shape), device))
