"""README's two snippets of a block between levels, run one after the other on the GPU, against the block's formula."""
import os

import pytest
import torch

from .conftest import ROOT
from .test_gpu_feed_forward_layers import CLOSE, DEV, _formula, _near

pytestmark = pytest.mark.gpu


def _snippet(title):
    section = open(os.path.join(ROOT, "README.md")).read().split("## " + title + "\n")[1].split("\n## ")[0]
    return "\n".join(line[4:] for line in section.splitlines() if line.startswith("    "))


class Names(dict):
    """What the snippets have at hand; `history`: the fine level's features, one after the other."""

    def __init__(self, **given):
        super().__init__(given)
        self.history = [given["fine_features"]]

    def __missing__(self, name):
        if name == "coarse_features":
            return torch.randn(self["coarse"].pts_.shape[0], self["coarse_channels"], device=DEV)
        raise KeyError(name)

    def __setitem__(self, name, value):
        super().__setitem__(name, value)
        if name == "fine_features":
            self.history.append(value)


def test_readme_counts_the_features_of_a_block_once():
    torch.manual_seed(6)
    points = torch.rand(900, 3, device=DEV)
    ids = torch.arange(900, device=DEV, dtype=torch.int32) // 450
    names = Names(points=points, batch_ids=ids, coarse_channels=24, fine_channels=48, torch=torch,
                  fine_features=torch.randn(900, 48, device=DEV))
    for title in ("Attention between two levels", "The feed-forward half of a block"):
        exec(_snippet(title), {}, names)
    given, attended, fed, served = names.history
    assert not torch.equal(given, attended)
    want = _formula(names["block"], attended.detach().double(), None)[0]
    assert _near(fed, want, CLOSE[torch.float32])
    # served in 8 bits on top of that: a few percent of the update
    total = fed.detach().double()
    update = _formula(names["block"], total, None)[0].detach() - total
    assert float((served.double() - total - update).norm()) <= 0.1 * float(update.norm())
