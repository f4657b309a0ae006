"""What of the kernel library's C ABI can be seen without the plugin and without a GPU."""
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_kernel_library_alone_exports_what_the_header_declares(pkg):
    code = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "b200_whisper.h")).read(), flags=re.S)      # declarations only
    names = sorted(set(re.findall(r"\b(b200_[a-z0-9_]+)\s*\(", code)))
    lib = pkg.kernels_lib()
    assert len(names) >= 20 and [n for n in names if not hasattr(lib, n)] == []
    assert b"sm_100a" in lib.b200_version()
