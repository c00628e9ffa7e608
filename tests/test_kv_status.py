"""What the K/V cache's kernels report must not hide a wait that ran out: that one restarts the exchange between ranks (no GPU needed)."""
import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nihilus_b200", "csrc")


def test_reports_of_the_cache_never_replace_an_exhausted_wait():
    seen = 0
    for path in glob.glob(os.path.join(CSRC, "*.cu*")):
        with open(path) as f:
            for line in f:
                if re.search(r"atomic\w+\(.*DEV_KV_", line):
                    seen += 1
                    assert re.search(r"atomicCAS\([\w.]*status, DEV_OK, DEV_KV_\w+\)", line), (os.path.basename(path), line.strip())
    assert seen >= 5
