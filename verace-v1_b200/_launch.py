"""The launch path of the decode step's small calls, where the host's share of a call is longer
than the kernel: the current stream's handle without the Python objects of
``torch.cuda.stream`` (``raw_stream(index)``), and the current device's index (``current()``)
to skip the device guard where it changes nothing."""
import torch

raw_stream = torch._C._cuda_getCurrentRawStream
current = torch._C._cuda_getDevice
