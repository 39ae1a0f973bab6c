"""The bench's recorded HBM bytes belong to the quantizer that it times, without a GPU."""

import json
import os

import bench

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_the_counter_pass_ran_on_the_current_quantizer_sources():
    """bench.py leaves roofline.traffic empty otherwise: after a change to a file of bench.QUANTIZER_SOURCES (the public
    header and the common ones among them) the passes of profiles/quant_c2_hbm_counters.md are run again."""
    with open(os.path.join(ROOT, "profiles", "quant_c2_traffic.json")) as f:
        record = json.load(f)
    assert record["quantizer_source_hash"] == bench.quantizer_source_hash()
    for role, per in (("key", bench.algorithmic_bytes(8, True, bench.LAYERS)),
                      ("value", bench.algorithmic_bytes(4, False, bench.LAYERS))):
        read, write = record[f"{role}_launch_read_bytes"], record[f"{role}_launch_write_bytes"]
        assert record[f"{role}_launch_bytes"] == read + write and record[f"{role}_algorithmic_bytes"] == per
        assert per <= read + write < 1.05 * per
    with open(os.path.join(ROOT, "profiles", "quant_c2_hbm_counters.md")) as f:
        assert record["quantizer_source_hash"] in f.read()
