"""bench.py reports the recorded HBM traffic only while it was counted on the present kernels: a change to one of their sources or headers takes the record again
(python3 bench.py --traffic --write-traffic --no-cpu) or loses the figure."""
import json
import os


def test_the_record_is_of_the_present_sources():
    import bench
    with open(os.path.join(bench.ROOT, "profiles", "ns_gemm_traffic.json")) as f:
        assert json.load(f)["source_sha16"] == bench.kernel_source_sha16()
