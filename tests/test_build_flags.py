"""`make check-hazards` scans the code that ships: every source with the flags its object is built with (dry runs, no compiler)."""
import os
import re
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _dry(*args):
    out = subprocess.run(["make", "-n", *args], cwd=ROOT, capture_output=True, text=True, check=True).stdout
    return out.replace("\\\n", " ").splitlines()


def _flags(words):
    return sorted(w for w in words if w.startswith("-f") and w != "-fPIC" or w.startswith("-D"))


def test_sources_are_scanned_with_their_own_flags():
    built = {}
    for line in _dry("-B"):
        m = re.search(r" -c (\S+\.hip) -o ", line)
        if m:
            assert "-packed-fp32-ops" in line
            built.setdefault(m.group(1), []).append(_flags(line.split()))
    scanned = {}
    for line in _dry("check-hazards"):
        m = re.search(r"hazard_scan\.py (\S+\.hip)(.*)", line)
        if m:
            assert "|" not in line, "a pipe hides the scan's status"
            scanned.setdefault(m.group(1), []).append(_flags(m.group(2).split()))
    assert {os.path.basename(f) for f in scanned} >= {"mpnn_beam.hip", "mpnn_optim.hip", "mpnn_edge.hip"}
    for source, flags in scanned.items():
        assert sorted(flags) == sorted(built[source]), source
    for source in set(built) - set(scanned):
        with open(os.path.join(ROOT, source)) as f:
            text = f.read()
        assert not re.search(r"\basm\b|mfma", text), f"{source} has assembly or matrix instructions and is not scanned"
