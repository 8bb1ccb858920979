"""The row operators of a head as torch operations on the host, so that its layers can be tested without a GPU."""
import torch

import head_oracle as oracle


class RowOperators:
    """What the compiled binding has under these names (seeds and offsets come signed)."""

    @staticmethod
    def layer_norm(x, weight, bias, eps):
        return torch.nn.functional.layer_norm(x, x.shape[-1:], weight, bias, eps)

    @staticmethod
    def dropout(x, p, seed, offset, state, residual):
        kept = oracle.keep(tuple(x.shape), p, seed % (1 << 64), offset % (1 << 64))
        out = torch.where(kept, x / (1 - p), torch.zeros(()))
        return out if residual is None else residual + out

    @classmethod
    def dropout_add_layer_norm(cls, x, residual, weight, bias, p, seed, offset, state, eps):
        h = cls.dropout(x, p, seed, offset, state, residual)
        return cls.layer_norm(h, weight, bias, eps), h
