"""Checks and the device guard that the model-side operators share."""
import torch

class _Nothing:
    def __enter__(self):
        pass

    def __exit__(self, *a):
        return False


_NONE = _Nothing()
_current = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def on_device_of(t):
    """Makes the tensor's device (and with it torch's current stream there) the current one for a call."""
    return _NONE if t.get_device() == _current() else torch.cuda.device(t.device)


def check_out(out, shape, dtype, device):
    if not (out.device == device and out.dtype == dtype and tuple(out.shape) == tuple(shape) and out.is_contiguous()):
        raise ValueError("out must be a contiguous %s tensor %s on %s" % (dtype, tuple(shape), device))
