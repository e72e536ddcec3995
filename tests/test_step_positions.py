"""The forms of a decode step's position (no GPU: a cache that keeps dense rows, the library's attention)."""
import importlib

import torch


class _Dense:
    def __init__(self):
        self.k = self.v = None

    def update_and_fetch(self, k, v):
        self.k = k if self.k is None else torch.cat([self.k, k], 2)
        self.v = v if self.v is None else torch.cat([self.v, v], 2)
        return self.k, self.v


def test_positions(tq):
    """One for the batch, as a tensor of one element or of none, or one per sequence."""
    q2 = importlib.import_module(tq.__name__ + ".qwen2")
    cfg = q2.Qwen2Config(n_layers=1, hidden=64, n_q_heads=2, n_kv_heads=1, ffn=64, vocab=50)
    model = q2.Qwen2Model(cfg, torch.device("cpu"), dtype=torch.float32)
    tok = torch.tensor([[3], [7]])
    want = model.decode_step(tok, [_Dense()], torch.tensor([5], dtype=torch.int32))
    for position in (torch.tensor(5, dtype=torch.int32), torch.tensor([5, 5], dtype=torch.int32), torch.tensor([[5], [5]])):
        assert torch.equal(model.decode_step(tok, [_Dense()], position), want)
