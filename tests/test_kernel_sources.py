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


EARLIER = re.compile(r"p\.positions\[|p\.block_table\[|[^_]table\[key|key_row\(p, (?!table, base)|to_float\(q\[|in_step\(p, |look_up\(item")


@pytest.mark.parametrize("name,kernel", [("attention_prefix.cu", "attention_prefix_simple_kernel"), ("attention_prefix.cu", "attention_prefix_mma_kernel"),
                                         ("attention_prefix.cu", "attention_prefix_merge_kernel"), ("attention_prefix_stream.cu", "attention_prefix_stream_kernel"),
                                         ("attention_prefix_tcgen05.cu", "attention_prefix_tc_kernel")])
def test_launches_of_shared_prefixes_look_before_they_read(name, kernel):
    """What the stream's earlier kernels wrote (positions, block tables, queries, the cache) is read behind begin_items or pass_gate alone."""
    text = (CSRC / name).read_text()
    body = text[re.search(rf"\n{kernel}\(", text).end():]
    looks = re.search(r"(begin_items|pass_gate)\(p\);\n(?!    if \(tid == 0\) atomicOr)", body)        # not the one of a CTA that gives up
    reads = EARLIER.search(body)
    assert looks and reads and looks.start() < reads.start()


def test_a_launch_that_did_not_wait_is_told_by_one_that_did():
    """Behind the first of a call's launches: an acquire of what the first released once it had waited, or a wait of its own."""
    text = (CSRC / "attention_prefix.cuh").read_text()
    begin = text[text.index("void begin_items("):]
    begin = begin[:begin.index("\n}")]
    assert re.search(r"if \(!p\.first\) \{[^}]*pass_gate\(p\);\s*return;", begin) and begin.index("pdl_wait();") < begin.index("open_gate(p);")
    assert "atom.release.gpu" in text and re.search(r"ld\.acquire\.gpu.*\n\s*if \(seen != p\.token\) pdl_wait\(\);", text)
    merge = (CSRC / "attention_prefix.cu").read_text()
    merge = merge[merge.index("attention_prefix_merge_kernel("):]
    assert merge.index("pdl_wait();") < merge.index("*p.gate = 0;")
