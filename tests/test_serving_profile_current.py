"""The committed profile of the serving kernels was taken on the sources in the tree."""

from __future__ import annotations

import re

from conftest import ROOT
from test_profiles_current import _bench


def test_serving_profile_records_the_current_sources():
    text = (ROOT / "profiles" / "serving_kernels.md").read_text()
    recorded = re.search(r"^serving source hash: `([0-9a-f]+)`", text, re.M)
    assert recorded and recorded.group(1) == _bench().kernel_source_hash(serving=True)
