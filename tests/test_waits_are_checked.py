"""Every wait of the tensor-core kernels is bounded; one that runs out must stop what relies on it. (No GPU test makes one
run out: that would take a broken kernel.)"""
from __future__ import annotations

import re
from pathlib import Path

CSRC = Path(__file__).resolve().parents[1] / "open-supersampling_b200" / "csrc"


def test_no_result_of_a_wait_is_dropped():
    for path in [*CSRC.glob("*.cu"), *CSRC.glob("*.cuh")]:
        for number, line in enumerate(path.read_text().splitlines(), 1):
            assert not re.match(r"\s*(tc::)?mbar_wait\(", line), f"{path.name}:{number}: {line.strip()}"


def test_blocks_count_a_wait_that_ran_out_in_any_of_their_threads():
    for name in ("attention_mma.cu", "attention_mma_bwd.cu"):
        assert not re.search(r"!alive && tid == 0\) count_timeout", (CSRC / name).read_text()), name
