"""Every command of the repository that compiles device code leaves packed f32 instructions out."""
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FLAG = "-Xclang -target-feature -Xclang -packed-fp32-ops"


def test_every_compile_command_has_the_flag():
    found = 0
    for folder, _, files in os.walk(ROOT):
        if os.path.relpath(folder, ROOT).split(os.sep)[0] not in (".", "speechrecognition_amd", "tools", "tests", "oracle"):
            continue
        for name in files:
            if not (name == "Makefile" or name.endswith((".sh", ".hip"))):
                continue
            text = open(os.path.join(folder, name), encoding="utf-8").read().replace("\\\n", " ")
            for line in re.findall(r".*(?:hipcc -|HIPCC\)|HIPFLAGS *:=).*", text):
                if "HIPFLAGS)" in line or "-shared" in line:
                    continue
                found += 1
                assert FLAG in line, (name, line)
    assert found >= 3


def test_build_compiles_what_is_built_already(monkeypatch):
    import subprocess
    import sys

    sys.path.insert(0, ROOT)
    import __graft_entry__ as entry
    from speechrecognition_amd import _capi
    commands = []
    monkeypatch.setattr(subprocess, "check_call", commands.append)
    monkeypatch.setattr(_capi, "load", lambda: None)
    entry.build()
    assert len(commands) == 3 and all("-B" in c for c in commands)
