"""__graft_entry__.build() makes the product (the kernels' library, the oracle, the import) whatever tests/cpp holds: a parity
driver of the C++ layer that is absent or does not build is reported, and its own tests say that it is not there."""
import shutil
import sys
import types
from pathlib import Path

import pytest

import __graft_entry__ as entry

REPO = Path(__file__).resolve().parent.parent
RULES = {
    "none": None,                                                       # no tests/cpp at all
    "one": "h3_kernels_test:\n\ttouch $@\n",                            # the other driver has no rule
    "broken": "h3_kernels_test:\n\ttouch $@\nh3_dense_test:\n\tfalse\n",  # and here it does not build
    "both": "h3_kernels_test h3_dense_test:\n\ttouch $@\n",
}


@pytest.mark.parametrize("kind", RULES)
def test_build_does_not_depend_on_the_test_drivers(kind, tmp_path, monkeypatch, capfd):
    (tmp_path / "oracle").mkdir()
    for f in (REPO / "oracle").iterdir():
        if f.suffix in (".c", ".h") or f.name == "Makefile":
            shutil.copy(f, tmp_path / "oracle")
    cpp = tmp_path / "tests" / "cpp"
    if RULES[kind] is not None:
        cpp.mkdir(parents=True)
        (cpp / "Makefile").write_text(RULES[kind])
        if kind == "broken":
            (cpp / "h3_dense_test").write_text("of an earlier build")
    built = []
    monkeypatch.setattr(entry, "REPO", tmp_path)
    monkeypatch.setattr(sys, "path", list(sys.path))
    monkeypatch.setitem(sys.modules, "build", types.SimpleNamespace(build=lambda: built.append("kernels")))
    entry.build()
    assert built == ["kernels"] and (tmp_path / "oracle" / "libmh3_oracle.so").exists()
    drivers = {"none": [], "one": ["h3_kernels_test"], "broken": ["h3_kernels_test"],
               "both": ["h3_kernels_test", "h3_dense_test"]}[kind]
    said = capfd.readouterr().err
    for name in ("h3_kernels_test", "h3_dense_test"):
        assert (cpp / name).exists() == (name in drivers)   # no driver of an earlier build stays in its place
        assert (f"{name}: not built" in said) == (name not in drivers)
