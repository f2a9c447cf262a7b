"""How the library is built: every object without packed FP32 instructions, and anew when the Makefile changes."""
import os
import re

MK = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "alphazero-connect6_amd", "csrc", "Makefile")).read()


def test_no_packed_fp32_anywhere():
    flags = re.search(r"^FLAGS := (.*)$", MK, re.M).group(1)
    assert "-Xclang -target-feature -Xclang -packed-fp32-ops" in flags
    assert "+packed-fp32-ops" not in MK
    assert all("$(FLAGS)" in line for line in re.findall(r"^\t.*-c \$<.*$", MK, re.M))


def test_objects_depend_on_the_makefile():
    assert re.search(r"^\$\(OUT\)/%\.o:.*\bMakefile\b", MK, re.M)


def test_build_compiles_every_time():
    import inspect

    import __graft_entry__ as g
    assert '"make", "-B"' in inspect.getsource(g.build)
