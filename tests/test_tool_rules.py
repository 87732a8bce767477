"""CPU: what the measuring tools may not hold.  A kernel variant that faulted is dropped, with its log as the record; no script
runs it again, and no switch is left whose use is to narrow a GPU fault down on the GPU."""
import os

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def sources(*tops):
    for top in tops:
        for folder, _, files in os.walk(os.path.join(ROOT, top)):
            for name in files:
                if name.endswith((".hip", ".hh", ".cc", ".h", ".sh", ".py")):
                    path = os.path.join(folder, name)
                    yield os.path.relpath(path, ROOT), open(path, errors="replace").read()


@pytest.mark.parametrize("phrase", ["QB_ONLY", "qb_A3", "qb_A4", "A3bar", "A3early", "in A4", "fault isolation"])
def test_no_tool_runs_a_faulting_variant_again(phrase):
    assert [p for p, text in sources("tools") if phrase in text] == []
