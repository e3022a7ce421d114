"""What the built library holds (no GPU)."""
import shutil
import subprocess

import pytest


def test_one_device_error_word(boa):
    """The word that kernels record a failure in is the one that the host
    reads: no object of the library holds a second one."""
    nm = shutil.which("nm")
    if nm is None:
        pytest.skip("needs binutils")
    names = subprocess.run([nm, "-C", boa.LIB_PATH], check=True, capture_output=True, text=True).stdout.splitlines()
    assert sum(x.endswith(" boa::g_dev_error") for x in names) == 1
