"""A cache of 8 bits on the host, straight from its definition: FP32 scales for 16 positions of a head, int8 codes."""

import torch

BLOCK = 16


class Blocks:
    """One sequence's codes [positions, heads, 64] and scales [blocks, heads], grown by appending FP16 values."""

    def __init__(self, heads):
        self.codes = torch.zeros(0, heads, 64, dtype=torch.float32)
        self.scales = torch.zeros(0, heads, dtype=torch.float32)

    def append(self, values):
        """values [tokens, heads, 64], as one call stores them."""
        if values.shape[0] == 0:
            return
        at, end = self.codes.shape[0], self.codes.shape[0] + values.shape[0]
        values = values.float().cpu()
        self.codes = torch.cat([self.codes, torch.zeros_like(values)])
        while self.scales.shape[0] * BLOCK < end:
            self.scales = torch.cat([self.scales, torch.zeros(1, self.codes.shape[1])])
        for block in range(at // BLOCK, -(-end // BLOCK)):
            first, last = max(at, block * BLOCK), min(end, (block + 1) * BLOCK)
            fresh = values[first - at:last - at]
            largest = fresh.abs().amax((0, 2))
            # (The quotient of two FP32 numbers in FP64, rounded to FP32, is their FP32 quotient.)
            scale = torch.where(largest <= 65504, (largest.double() / 127).float(), float("nan"))
            if first > block * BLOCK:
                scale = torch.maximum(scale, self.scales[block])      # keeps a NaN
                kept = self.codes[block * BLOCK:first]
                self.codes[block * BLOCK:first] = self.rounded(kept * self.scales[block][:, None], scale)
            self.codes[first:last] = self.rounded(fresh, scale)
            self.scales[block] = scale

    @staticmethod
    def rounded(values, scale):
        quotient = (values.double() / scale.double()[:, None]).float()
        return torch.where(scale[:, None] > 0, torch.round(quotient), 0.0)

    def values(self):
        """What the codes stand for, in FP64."""
        return self.codes.double() * self.scales.double().repeat_interleave(BLOCK, 0)[:self.codes.shape[0], :, None]
