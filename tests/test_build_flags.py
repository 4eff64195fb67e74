"""An object built with other compiler flags is out of date (seed_amd/build.py, tools/calib), with a compiler that only writes its output."""
import os
import stat

import pytest

from seed_amd import build as B
from tools import calib


@pytest.fixture
def compiler(tmp_path, monkeypatch):
    """A stand-in for hipcc: records the call, writes the output file, fails where the command holds -DFAIL."""
    path = tmp_path / "hipcc"
    path.write_text('#!/bin/sh\necho "$@" >> "%s"\ncase "$*" in *-DFAIL*) exit 1;; esac\nwhile [ $# -gt 0 ]; do [ "$1" = -o ] && echo built > "$2"; shift; done\n'
                    % (tmp_path / "calls"))
    path.chmod(path.stat().st_mode | stat.S_IXUSR)
    monkeypatch.setattr(B, "HIPCC", str(path))
    monkeypatch.setattr(calib, "HIPCC", str(path))
    return lambda: (tmp_path / "calls").read_text().count("\n") if (tmp_path / "calls").exists() else 0


def test_an_object_is_rebuilt_when_its_flags_change(compiler, tmp_path, monkeypatch):
    src = "kv_cache.hip"
    built = lambda *extra, force=False: B._compile(src, force, str(tmp_path), extra)[1]  # noqa: E731
    assert built() and not built() and compiler() == 1
    assert built("-DA") and not built("-DA") and built()                           # other extra flags, and back
    monkeypatch.setattr(B, "FLAGS", B.FLAGS + ["-ffast"])
    assert built() and not built() and built(force=True)


def test_an_object_without_a_record_or_from_a_failed_build_is_out_of_date(compiler, tmp_path):
    obj = tmp_path / "kv_cache.o"
    obj.write_text("from an earlier build")                                        # newer than its source, flags unknown
    assert B._compile("kv_cache.hip", False, str(tmp_path)) == (str(obj), True)
    with pytest.raises(RuntimeError, match="hipcc failed"):
        B._compile("kv_cache.hip", False, str(tmp_path), ("-DFAIL",))
    assert B._compile("kv_cache.hip", False, str(tmp_path))[1]
    assert not B._compile("kv_cache.hip", False, str(tmp_path))[1]


def test_the_calibration_library_is_rebuilt_without_a_record(compiler, tmp_path, monkeypatch):
    lib = tmp_path / "libseedcal.so"
    monkeypatch.setattr(calib, "LIB", str(lib))
    lib.write_text("from an earlier build")
    calib.build()
    assert compiler() == 1 and lib.read_text() == "built\n"
    calib.build()
    assert compiler() == 1
    os.remove(str(lib) + ".cmd")
    calib.build()
    assert compiler() == 2
