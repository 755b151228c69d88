"""The library's makefile: what a change of it, of a header or of a source builds again (make's own plan; nothing is compiled)."""
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ralf_amd", "csrc")


def compiled_after(changed):
    """the sources that make would compile if `changed` were new"""
    plan = subprocess.run(["make", "-n", "-W", changed], cwd=CSRC, check=True, capture_output=True, text=True).stdout
    words = [line.split() for line in plan.splitlines() if " -c " in line]
    return {w[w.index("-c") + 1] for w in words}


def sources():
    return {f for f in os.listdir(CSRC) if f.endswith(".hip")} | {"error.cpp"}


def test_flags_reach_every_unit():
    """the flags stand in the makefile: a change of it compiles all sources again, whatever objects are lying there"""
    assert compiled_after("Makefile") == sources()


@pytest.mark.parametrize("header", sorted(f for f in os.listdir(CSRC) if f.endswith(".h")))
def test_headers_reach_their_units(header):
    users, names = set(), {header}
    while True:         # what includes it, by itself or through another header
        more = {f for f in os.listdir(CSRC) if f.endswith((".hip", ".h", ".cpp")) and any(f'#include "{n}"' in open(os.path.join(CSRC, f)).read() for n in names)}
        if more <= names | users:
            break
        names |= {f for f in more if f.endswith(".h")}
        users |= {f for f in more if not f.endswith(".h")}
    assert users and users <= compiled_after(header)
