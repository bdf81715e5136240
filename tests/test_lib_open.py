"""Opening a library that is not this package's own build."""
import subprocess

import pytest

from eval_driving_safety_amd import _lib


@pytest.mark.parametrize("source", ["int adv_abi_version(void) { return 11; }", "int adv_abi_version(void) { return 3; }", "int other;"])
def test_a_stale_build_is_named_as_one(tmp_path, source):
    (tmp_path / "old.c").write_text(source)
    subprocess.run(["gcc", "-shared", "-fPIC", "-o", str(tmp_path / "libold.so"), str(tmp_path / "old.c")], check=True)
    with pytest.raises(ImportError, match="libold.so .* - rebuild"):
        _lib._open(str(tmp_path / "libold.so"))
