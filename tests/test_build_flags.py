"""How the extension is compiled."""
import os
import runpy

import setuptools

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_stand_in_headers_come_last(monkeypatch):
    """csrc/compat declares a class of another library for a header that torch
    may come to ship: it must not be found before that one."""
    seen = {}
    monkeypatch.setattr(setuptools, "setup", lambda **kw: seen.update(kw))
    monkeypatch.chdir(REPO)
    runpy.run_path(os.path.join(REPO, "setup.py"))
    ext, = seen["ext_modules"]
    assert not any("compat" in d for d in ext.include_dirs)
    flags = ext.extra_compile_args["cxx"]
    at = flags.index("-idirafter")
    assert os.path.isdir(os.path.join(flags[at + 1], "nlohmann"))
