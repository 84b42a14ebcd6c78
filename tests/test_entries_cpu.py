"""The C entry points of the mixture and the head throw nothing: each one's calls into the
library stand inside the functions that catch (read from the source: only running out of
host memory would show it)."""

import re

from conftest import ROOT

SOURCE = (ROOT / "macboost_b200" / "csrc" / "capi.cpp").read_text()
NAMES = ["route_device", "route_grad_device", "sort_rows_workspace", "sort_rows_device",
         "gather_rows_device", "combine_rows_device", "combine_rows_grad_device", "head_workspace",
         "head_loss_device", "head_grad_device", "head_check_device"]


def test_calls_are_guarded():
    for name in NAMES:
        at = SOURCE.index(f"macboost_{name}(")
        body = SOURCE[at:SOURCE.index("\n}\n", at)]
        call = re.search(r"return guarded(_size)?\((err, )?\[&\].*mb::" + name + r"\(", body, re.S)
        assert call and body.count("mb::" + name) == 1, name
