"""Shared-memory layouts of the tensor-core attention over the INT8 cache, read
from the sources' constants: the word that every thread reads its TMEM address
from, after the setup barrier, lies behind the barriers and before whatever is
written from then on."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "qwen-image-2.1-accel_b200" / "csrc"


def constants(*names):
    """The files' integer constants, by name."""
    got = {}
    for name in names:
        for decl in re.findall(r"^constexpr int ([^;{()]*=[^;{]*);", (CSRC / name).read_text(), re.M):
            for item in decl.split(","):
                left, right = item.split("=", 1)
                got[left.strip()] = eval(right.replace("/", "//"), {}, got)
    return got


@pytest.mark.parametrize("name,following", [("cached_attn_tiles.cu", "kSmemStage"), ("cached_attn_wide.cu", None)])
def test_tmem_address_has_a_place_of_its_own(name, following):
    text = (CSRC / name).read_text()
    c = constants("cached_attn.cuh", "cached_attn_tc.cuh", name)
    place = re.search(r"tmem_slot = reinterpret_cast<uint32_t\*>\((\w+) \+ (\w+)\)", text)
    start = eval(place[2], {}, c)
    if place[1] == "bars":                          # counted in barriers
        start = c["kSmemBars"] + 8 * start
    last = max(int(i) for i in re.findall(r"= bars \+ (\d+);", text))
    end = c[following] if following else c["kSmemBytes"] - 1024     # (1 KB of alignment)
    assert c["kSmemBars"] + 8 * (last + 1) <= start and start + 4 <= end
    assert c["kSmemBytes"] <= 227 * 1024
