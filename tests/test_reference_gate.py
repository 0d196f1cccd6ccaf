"""The engine drop-in tests may skip only where the build had no reference; a built library that got lost on the way fails them."""
import os
import shutil
import subprocess

import pytest

from conftest import ROOT, reference_expected


def make_ref(tree, reference="/nonexistent"):
    shutil.copy(os.path.join(ROOT, "oracle", "Makefile"), os.path.join(tree, "oracle", "Makefile"))
    subprocess.run(["make", "-s", "-C", os.path.join(tree, "oracle"), "ref", f"REF_ROOT={reference}"], check=True, capture_output=True)


@pytest.fixture
def tree(tmp_path):
    if shutil.which("make") is None:
        pytest.skip("no make")
    (tmp_path / "oracle").mkdir()
    return str(tmp_path)


def test_without_a_reference_the_tests_may_skip(tree):
    make_ref(tree)
    assert not reference_expected(tree)


def test_a_library_that_did_not_travel_is_missed(tree):
    os.mkdir(os.path.join(tree, "oracle", "_ref"))
    open(os.path.join(tree, "oracle", "_ref", "libnvk_ref_dropin.so"), "w").close()
    make_ref(tree)
    assert reference_expected(tree)
    shutil.rmtree(os.path.join(tree, "oracle", "_ref"))  # the folder as a whole, as when a snapshot leaves it out
    assert reference_expected(tree)


def test_a_tree_that_was_never_built_is_missed(tree):
    assert reference_expected(tree)
