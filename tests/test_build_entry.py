"""The build entry on test folders other than this one: the product is built first, and of the tests' helpers what is there."""
import sys

import pytest

import __graft_entry__ as entry

FILE = """
built = []
def build(force=False): built.append("build")
def build_library(force=False): built.append("build_library")
"""


@pytest.fixture
def no_module(monkeypatch):
    monkeypatch.delitem(sys.modules, "emu_gen_sources", raising=False)
    yield
    sys.modules.pop("emu_gen_sources", None)


def test_helpers_that_are_not_there_are_left_out(tmp_path, no_module):
    path = tmp_path / "gen_sources.py"
    path.write_text(FILE)
    assert entry.build_test_helpers(str(path)) == ["build", "build_library"] == sys.modules["emu_gen_sources"].built


def test_no_tests_folder(tmp_path, no_module):
    assert entry.build_test_helpers(str(tmp_path / "gen_sources.py")) == []


def test_this_folder_offers_all_of_them(emu_sources):
    assert [name for name in entry.TEST_HELPERS if not hasattr(emu_sources, name)] == []


def test_a_helper_that_fails_is_not_passed_over(tmp_path, no_module):
    path = tmp_path / "gen_sources.py"
    path.write_text("def build(force=False): raise SystemExit('an edit no longer applies')\n")
    with pytest.raises(SystemExit, match="no longer applies"):
        entry.build_test_helpers(str(path))


def test_the_product_comes_first(monkeypatch, tmp_path):
    """Nothing of a tests folder is touched before the library is built and looked at."""
    order = []

    class Builder:
        @staticmethod
        def build(verbose=False):
            order.append("library")

    monkeypatch.setitem(sys.modules, entry.PKG_NAME + "_build", Builder)
    monkeypatch.setattr(entry.subprocess, "run", lambda *a, **kw: order.append("oracle"))
    monkeypatch.setattr(entry, "build_cpp_tests", lambda: order.append("programs"))
    monkeypatch.setattr(entry, "build_test_helpers", lambda: order.append("helpers") or [])
    entry.build()
    assert order == ["library", "oracle", "programs", "helpers"]
