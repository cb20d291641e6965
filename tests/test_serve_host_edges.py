"""The serving operators without a device, at their edges."""

from __future__ import annotations

import re

from conftest import ROOT

CSRC = ROOT / "delta_feedback_experiment_amd" / "csrc"


def test_lane_reads_are_widened_without_their_sign():
    """The lane reads return int: in a 64-bit mask a word with its top bit set
    would fill the upper word, and name keys past the sequence."""
    found = 0
    for path in sorted((CSRC / "serve").glob("*")):
        for statement in path.read_text().split(";"):
            if "uint64_t" not in statement or "<< 32" not in statement:
                continue
            for m in re.finditer(r"__builtin_amdgcn_read(?:first)?lane\(", statement):
                found += 1
                assert statement[:m.start()].endswith("(uint32_t)"), (path.name, statement.strip())
    assert found
