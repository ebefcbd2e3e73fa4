"""bench.py quotes the committed profiles of the train step as long as the step's own kernel sources stand."""
import os
import shutil

import bench
from midiemo.build import CSRC, STEP_SOURCES


def test_the_hash_follows_the_sources_of_the_step_alone(tmp_path, monkeypatch):
    there = tmp_path / "midi-emotion_amd" / "csrc"
    there.mkdir(parents=True)
    for n in os.listdir(CSRC):
        if n.endswith((".hip", ".h")):
            shutil.copy(os.path.join(CSRC, n), there / n)
    first = bench.source_hash()
    monkeypatch.setattr(bench, "ROOT", str(tmp_path))
    assert bench.source_hash() == first
    (there / "me_new.hip").write_text("// kernels of something else\n")
    with open(there / "me_decode.hip", "a") as f:
        f.write("\n// another line\n")
    assert bench.source_hash() == first
    for n in STEP_SOURCES:
        text = (there / n).read_text()
        (there / n).write_text(text + "\n// another line\n")
        assert bench.source_hash() != first, n
        (there / n).write_text(text)
    assert bench.source_hash() == first
