"""splat_labels.h states the limits that the library holds to."""

from __future__ import annotations

import re
from pathlib import Path

ROOT = Path(__file__).resolve().parents[1]

HEADER = " ".join(re.sub(r"\n \*", " ", (ROOT / "include/splat_labels.h").read_text()).split())


def test_the_header_states_the_limits_that_are_checked():
    sources = {name: (ROOT / "splatting-rs_b200/csrc" / name).read_text() for name in ("embedding.cu", "label_head.cu")}
    assert all("dim < (1u << 20)" in text for text in sources.values())
    assert "entries below 2^31, dim below 2^20" in HEADER
    assert "labels are below 2^31 - 512, dim below 2^20" in HEADER


def test_the_header_asks_for_the_normalizers_of_the_same_handle():
    assert "`d_log_normalizers` are those of this handle's sp_label_head_loss" in HEADER
