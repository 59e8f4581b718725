"""Host -> device transfers that do not stall the host.

A pageable host tensor copied to the GPU makes the host wait for the copy, and the copy
waits for the work already queued on the stream: inside a forward that drains the whole
queue, after which the GPU idles while the host enqueues the next launches.  ``to_device``
stages a small host array in pinned memory and copies it with ``non_blocking=True`` on the
current stream (torch's caching host allocator keeps a pinned block until the copies that
read it have run, so the staging tensor may be dropped at once).  For a CPU device it is a
plain tensor.

A graph that is being captured would record that copy and read the staging memory again at every
replay, when it holds something else: host values are refused there.  Device tensors made before the
capture, and written between replays, take their place.
"""

from __future__ import annotations

import torch


def to_device(values, dtype: torch.dtype, device) -> torch.Tensor:
    """values (a list / nested list, or a CPU tensor) as a dtype tensor on device; not while the
    current stream is captured."""
    device = torch.device(device)
    if device.type == "cuda" and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("host values cannot be uploaded while a graph is captured (a replay would "
                           "read their staging memory again): give a tensor on the device")
    if isinstance(values, torch.Tensor):
        host = values.to(dtype=dtype)
        if device.type != "cuda":
            return host.to(device)
        return host.contiguous().pin_memory().to(device, non_blocking=True)
    if device.type != "cuda":
        return torch.tensor(values, dtype=dtype, device=device)
    return torch.tensor(values, dtype=dtype, pin_memory=True).to(device, non_blocking=True)
