"""Rules of synchronisation that show in no result a test could rely on, read from the sources."""
import glob
import os
import re

from conftest import ROOT

CSRC = os.path.join(ROOT, "moe-explore_b200", "csrc")


def _sources():
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu*"))):
        with open(path) as f:
            yield os.path.basename(path), re.sub(r"//[^\n]*", "", f.read())


def test_every_arrival_releases():
    """What a barrier guards changes hands by arrivals that release (the default): nobody is let on by one that orders nothing."""
    arrivals = [(name, a) for name, text in _sources() for a in re.findall(r"mbarrier\.arrive[\w.:]*", text)]
    assert len(arrivals) >= 4
    assert [x for x in arrivals if "relaxed" in x[1]] == []
