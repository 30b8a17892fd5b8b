# -*- coding: utf-8 -*-
"""What the build does besides compiling."""

import importlib.util
import os

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _setup():
    spec = importlib.util.spec_from_file_location(
        "stoke_setup", os.path.join(REPO, "setup.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def test_objects_older_than_a_header_are_compiled_again(tmp_path):
    folder = tmp_path / "temp" / "csrc"
    folder.mkdir(parents=True)
    header, old, new, other = (
        tmp_path / "x.h", folder / "a.o", folder / "b.o", folder / "a.txt")
    for i, f in enumerate((old, other, header, new)):
        f.write_text("")
        os.utime(f, (1000 + i, 1000 + i))
    _setup().drop_old_objects(str(tmp_path / "temp"), [str(header)])
    assert not old.exists() and new.exists() and other.exists()
    _setup().drop_old_objects(str(tmp_path / "absent"), [str(header)])


def test_build_lists_every_source_and_header():
    text = open(os.path.join(REPO, "setup.py")).read()
    for name in os.listdir(os.path.join(REPO, "csrc")):
        if name.endswith((".hip", ".h")):
            assert f"csrc/{name}" in text, name
