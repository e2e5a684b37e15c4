"""What the kernels' sources have to hold where a run cannot show it (host only): orders between kinds of memory accesses."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "sprout_lm_b200" / "csrc"
# a ring in shared memory that TMA fills and tcgen05 products read, cleared (wholly or by rows) with ordinary stores
CLEARS = re.compile(r"\(\(uint4\*\)s[KV]\)\[i\] = make_uint4\(0, 0, 0, 0\);|\*\(uint4\*\)\(sV \+ [^;]*= make_uint4\(0, 0, 0, 0\);")


@pytest.mark.parametrize("name", ["attention_tcgen05.cu", "attention_maps_tcgen05.cu", "attention_prefix_tcgen05.cu"])
def test_cleared_stages_are_fenced_before_anyone_is_told(name):
    """Ordinary stores and the asynchronous proxy (TMA writes, tcgen05 reads) are ordered by a proxy fence of the thread that stored, ahead of
    the barrier behind which the other side goes on."""
    text = (CSRC / name).read_text()
    clears = list(CLEARS.finditer(text))
    assert clears
    for clear in clears:
        told = re.search(r"__syncthreads\(\)|mbar_arrive\(", text[clear.end():])
        assert "fence_proxy_async();" in text[clear.end():clear.end() + told.start()]
