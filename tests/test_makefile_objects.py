"""Every source of the native engine has an object in the library, and every object is rebuilt
when a header that its source includes changes."""
import glob
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "persistentkv-attention_amd", "csrc")
SOURCES = sorted(os.path.basename(p) for p in glob.glob(os.path.join(CSRC, "*.hip")))


def _rules():
    with open(os.path.join(CSRC, "Makefile")) as f:
        return f.read().replace("\\\n", " ")


@pytest.mark.parametrize("source", SOURCES)
def test_objects_follow_their_headers(source):
    target = source.replace(".hip", ".o")
    rules = _rules()
    with open(os.path.join(CSRC, source)) as f:
        headers = re.findall(r'^#include "([^"]+)"', f.read(), re.M)
    needs = re.search(rf"^{re.escape(target)}:(.*)$", rules, re.M).group(1).split()
    assert source in needs and "pkv.h" in headers
    for h in headers:
        assert h in needs or f"$(INC)/{h}" in needs, f"{target} does not depend on {h}"
    assert target in re.search(r"^OBJECTS\s*:=(.*)$", rules, re.M).group(1).split()


def test_the_library_links_the_objects():
    out = subprocess.run(["make", "-n", "-B", "PYTHON=true", "../libpkv.so"], cwd=CSRC, capture_output=True, text=True)
    link = [line for line in out.stdout.splitlines() if "-shared" in line][-1]
    assert all(s.replace(".hip", ".o") in link for s in SOURCES)
