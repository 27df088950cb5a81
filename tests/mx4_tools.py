"""Microscaled 4-bit numbers and expert layers in plain float64, for the tests."""
import math

import torch

GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
EVEN = (True, False, True, False, True, False, True, False)      # whose mantissa bit is 0


def quantized(x):
    """The values (float64) that x [..., width] becomes, and the scale bytes, one number at a time."""
    flat = x.double().reshape(-1, x.shape[-1]).tolist()
    values, scales = [], []
    for row in flat:
        out, marks = [], []
        for at in range(0, len(row), 32):
            block = row[at:at + 32]
            if any(not math.isfinite(v) for v in block):
                out += [math.nan] * len(block)
                marks.append(255)
                continue
            top = max(abs(v) for v in block)
            s = min(254, max(0, math.frexp(top)[1] - 1 - 2 + 127)) if top else 0
            marks.append(s)
            for v in block:
                size = min(6.0, abs(v) * 2.0 ** (127 - s))
                q = min(range(8), key=lambda i: (abs(GRID[i] - size), not EVEN[i]))
                out.append(math.copysign(GRID[q], v) * 2.0 ** (s - 127))
        values.append(out)
        scales.append(marks)
    return torch.tensor(values, dtype=torch.float64).reshape(x.shape), torch.tensor(scales)


def packed(values, marks):
    """values [rows, width] of the grid times 2^(marks - 127) -> (codes, scales) uint8 on the CPU, bit by bit."""
    rows, width = values.shape
    groups = -(-width // 128)
    codes = torch.zeros((rows, 64 * groups), dtype=torch.uint8)
    scales = torch.zeros((rows, 4 * groups), dtype=torch.uint8)
    for r in range(rows):
        words = [0] * (16 * groups)
        for k in range(width):
            s = int(marks[r, k // 32])
            scales[r, k // 32] = s
            v = float(values[r, k])
            if s == 255:
                continue
            code = GRID.index(abs(v) * 2.0 ** (127 - s)) | (8 if math.copysign(1.0, v) < 0 else 0)
            group, b, e = k // 128, k % 128 // 32, k % 32
            t, i = e // 8, e % 8
            words[16 * group + 4 * t + b] |= code << (4 * (i // 2) + 16 * (i % 2))
        for i, word in enumerate(words):
            for byte in range(4):
                codes[r, 4 * i + byte] = word >> (8 * byte) & 255
    return codes, scales


def activation(z, name):
    if name == "gelu_new":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    if name == "gelu":
        return 0.5 * z * (1 + torch.erf(z / math.sqrt(2)))
    if name == "relu2":
        return torch.relu(z) ** 2
    return torch.tanh(z) if name == "tanh" else z


def gated(gate, up, limit, alpha, form):
    if form == "silu":
        return gate * torch.sigmoid(gate) * up
    if form == "gelu_tanh":
        return activation(gate, "gelu_new") * up
    g = torch.clamp(gate, max=limit)
    return g * torch.sigmoid(alpha * g) * (torch.clamp(up, -limit, limit) + 1)
