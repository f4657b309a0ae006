"""The smoke entry point where the driver over whisper.h was left out of the build."""
import pytest

pytestmark = pytest.mark.gpu


def test_smoke_of_the_kernel_library_alone(pkg, capsys):
    import __graft_entry__ as entry
    entry._smoke_kernels(pkg)
    assert "kernel launches" in capsys.readouterr().out
