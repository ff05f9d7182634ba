"""The Python side of the shared-prefix attention's plan, without a GPU."""
import pytest
import torch

from mod_b200.ops import native as N


class Fake:
    """Stands for the extension: sizes as asked for, a plan that can be refused."""

    def __init__(self):
        self.refuse = False

    def attn_shared_sizes(self, T, B, G, Hq, Hkv, D, width, device):
        return 64, 32 * T

    def attn_shared_plan(self, *args):
        if self.refuse:
            raise RuntimeError("refused")


def test_a_refused_plan_stays_the_earlier_one(monkeypatch):
    fake = Fake()
    monkeypatch.setattr(N, "_C", lambda: fake)
    i = lambda n: torch.zeros(n, dtype=torch.int32)  # noqa: E731
    p = N.attn_shared_plan(torch.zeros(8, 3, dtype=torch.int32), i(8), i(3), i(2), 8, 16, 4, 128)
    said = {k: getattr(p, k) for k in p.__slots__}
    assert said["q_shape"] == (8, 16, 128) and said["groups"] == 2 and said["kv_heads"] == 4
    fake.refuse = True
    with pytest.raises(RuntimeError, match="refused"):
        N.attn_shared_plan(torch.zeros(4, 2, dtype=torch.int32), i(4), i(2), i(1), 4, 8, 2, 64, plan=p)
    assert all(getattr(p, k) is said[k] or getattr(p, k) == said[k] for k in said if k != "buf") and p.buf is said["buf"]
    # so that what was made for the refused sizes is told apart
    with pytest.raises(ValueError, match="other shapes"):
        N.attn_shared(torch.zeros(4, 8, 64), torch.zeros(2, 2, 16, 64), torch.zeros(2, 2, 64, 16),
                      torch.zeros(4, 2, dtype=torch.int32), p)
    fake.refuse = False
    again = N.attn_shared_plan(torch.zeros(4, 2, dtype=torch.int32), i(4), i(2), i(1), 4, 8, 2, 64, plan=p)
    assert again is p and p.q_shape == (4, 8, 64) and p.groups == 1 and p.table_shape == (4, 2) and p.ws_elems == 128
