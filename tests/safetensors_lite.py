"""Reading and writing whole float32 safetensors files, for tests that change a model folder's tensors."""
import json
import struct

import numpy as np
import torch


def load(path):
    with open(path, "rb") as fh:
        n = struct.unpack("<Q", fh.read(8))[0]
        head, body = json.loads(fh.read(n)), fh.read()
    out = {}
    for name, e in head.items():
        if name == "__metadata__":
            continue
        assert e["dtype"] == "F32"
        lo, hi = e["data_offsets"]
        out[name] = torch.from_numpy(np.frombuffer(body[lo:hi], np.float32).copy()).view(*e["shape"])
    return out


def save(path, tensors):
    head, at = {}, 0
    for name, t in tensors.items():
        head[name] = {"dtype": "F32", "shape": list(t.shape), "data_offsets": [at, at + 4 * t.numel()]}
        at += 4 * t.numel()
    raw = json.dumps(head).encode()
    raw += b" " * (-len(raw) % 8)
    with open(path, "wb") as fh:
        fh.write(struct.pack("<Q", len(raw)) + raw)
        for t in tensors.values():
            fh.write(t.contiguous().numpy().tobytes())
