"""The DRAM traffic records under profiles/ belong to the sources they name: bench.py prints a kernel's
traffic only while its source file is the one that was captured, so a change there needs a new capture."""

import glob
import json
import os

import pytest

import bench

RECORDS = sorted(glob.glob(os.path.join(bench.ROOT, "profiles", "*.json")))


@pytest.mark.parametrize("path", RECORDS, ids=os.path.basename)
def test_record_is_of_the_present_source(path):
    rec = json.load(open(path))
    assert rec["source_sha1"] == bench.source_sha(rec["source"])
    traffic, _ = bench.profiled_traffic(os.path.basename(path)[: -len(".json")])
    assert traffic == rec["dram_bytes_per_launch"] == rec["dram_bytes_read"] + rec["dram_bytes_write"]


def test_there_are_records():
    assert RECORDS
