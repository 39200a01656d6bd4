"""The counter record that the benchmark's line reports as measured traffic."""
import json
import os
import re

import bench


def test_the_record_is_of_these_sources():
    """The record of the dominant launch's HBM traffic holds the hash of the sources
    that its kernel is compiled from: a change to one of them needs the two counter
    runs of its document again."""
    rec = json.load(open(bench.TRAFFIC_FILE))
    assert rec["source_sha256"] == bench.kernel_source_hash()
    traffic, note = bench.measured_traffic(rec["launch"], rec["copies"])
    assert traffic == rec["fetch_bytes"] + rec["write_bytes"], note
    text = open(os.path.join(bench.ROOT, rec["source"])).read()
    assert rec["source_sha256"] in text and f"{rec['fetch_bytes']:,}" in text


def test_the_hash_covers_what_the_kernel_includes_and_nothing_else():
    """The kernel's source file and every header it includes, directly or not: edits of
    other files do not make the record another build's."""
    csrc = os.path.join("aiimage_amd", "csrc")
    seen, left = set(), ["aexq_qmv_q4.hip"]
    while left:
        name = left.pop()
        if name not in seen:
            seen.add(name)
            text = open(os.path.join(bench.ROOT, csrc, name)).read()
            left += re.findall(r'#include "([^"]+)"', text)
    assert sorted(bench.KERNEL_SOURCES) == sorted(os.path.join(csrc, n) for n in seen)
