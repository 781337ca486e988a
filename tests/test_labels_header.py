"""splat_labels.h states the limits that the library holds to."""

from __future__ import annotations

import re
from pathlib import Path

ROOT = Path(__file__).resolve().parents[1]


def test_the_header_states_the_limits_that_are_checked():
    header = " ".join(re.sub(r"\n \*", " ", (ROOT / "include/splat_labels.h").read_text()).split())
    sources = {name: (ROOT / "splatting-rs_b200/csrc" / name).read_text() for name in ("embedding.cu", "label_head.cu")}
    assert all("dim < (1u << 20)" in text for text in sources.values())
    assert "entries below 2^31, dim below 2^20" in header
    assert "labels are below 2^31 - 512, dim below 2^20" in header
