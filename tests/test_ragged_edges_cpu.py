"""Calls at the edges of the ragged expert path, on the CPU: arguments that do not go
together, no tokens, weights of little mass, derivatives that the operators do not have."""
import pytest
import torch

from learning_at_home_amd.ops import functional as Fops
from learning_at_home_amd.ops import ragged


def layout_of(ids, E):
    return Fops.ragged_layout(torch.tensor(ids, dtype=torch.int32), E)


class TestRowsRefuse:
    layout = layout_of([[0, 2], [2, 1], [-1, 1]], 3)
    x, y, w = torch.zeros(3, 8), torch.zeros(6, 8), torch.ones(3, 2)

    @pytest.mark.parametrize("change,match", [
        (dict(x=torch.zeros(2, 8)), "x must be"),  # fewer tokens than the layout's
        (dict(x=torch.zeros(4, 8)), "x must be"),
        (dict(x=torch.zeros(3)), "x must be"),
        (dict(x=torch.zeros(3, 8, device="meta")), "one device"),
        (dict(rows=layout.rows.long()), "int32"),
        (dict(order=layout.order.long()), "int32"),
        (dict(order=layout.order[:4]), "order"),
        (dict(rows=layout.rows.flatten()), "rows"),
    ])
    def test_gather(self, change, match):
        change = dict(change)
        x = change.pop("x", self.x)
        with pytest.raises(ValueError, match=match):
            Fops.ragged_gather(x, self.layout._replace(**change))

    @pytest.mark.parametrize("change,match", [
        (dict(y=torch.zeros(5, 8)), "y must be"),
        (dict(y=torch.zeros(6)), "y must be"),
        (dict(y=torch.zeros(6, 8, device="meta")), "one device"),
        (dict(weights=torch.ones(3, 1)), "weights must be"),  # would be read as [3, 2]
        (dict(weights=torch.ones(2, 2)), "weights must be"),
        (dict(weights=torch.ones(6)), "weights must be"),
        (dict(weights=torch.ones(3, 2, device="meta")), "one device"),
        (dict(layout=layout._replace(order=layout.order[:4])), "order"),
    ])
    def test_combine(self, change, match):
        with pytest.raises(ValueError, match=match):
            Fops.ragged_combine(**{**dict(y=self.y, layout=self.layout, weights=self.w), **change})

    @pytest.mark.parametrize("y,match", [(torch.zeros(5, 8), "y must be"), (torch.zeros(6), "y must be"),
                                         (torch.zeros(6, 8, device="meta"), "one device")])
    def test_ungather(self, y, match):
        with pytest.raises(ValueError, match=match):
            Fops.ragged_ungather(y, self.layout)

    @pytest.mark.parametrize("t,match", [(torch.zeros(3, 8), "bf16"), (torch.zeros(3, 8).half(), "bf16"),
                                         (torch.zeros(3, 12).bfloat16(), "multiple of 8")])
    def test_what_the_kernels_do_not_take(self, t, match):
        with pytest.raises(ValueError, match=match):
            ragged._check_gpu_rows(t, "x")
