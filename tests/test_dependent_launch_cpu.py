"""Kernels that may start before the kernel ahead of them in the stream has ended (gridDependencyWait) read global memory by ordinary loads only.

A non-coherent load (ld.global.nc, __ldg, a plain read through a `const __restrict__` parameter) promises that nobody writes the data while the kernel runs. The
kernel ahead does, until the wait ends; with that promise the compiler may move the load in front of the wait, and it has. Read from the sources, since whether
a build shows it depends on how the compiler schedules each kernel."""
import re
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "tensorrt_b200" / "csrc"
FILES = sorted(CSRC.glob("*.cu")) + sorted(CSRC.glob("*.cuh"))


def _code(path):
    return re.sub(r"//[^\n]*", "", path.read_text())


def _kernels(text):
    """(name, parameters, body) of each __global__ function."""
    for m in re.finditer(r"__global__\s+void\s", text):
        i = m.end()
        while True:  # attributes in parentheses before the name, then the parameters
            name = re.compile(r"\s*(\w+)\s*\(").match(text, i)
            depth, j = 1, name.end()
            while depth:
                depth += {"(": 1, ")": -1}.get(text[j], 0)
                j += 1
            if not name[1].startswith("__"):
                break
            i = j
        params = text[name.end():j - 1]
        j = text.index("{", j)
        depth, k = 1, j + 1
        while depth:
            depth += {"{": 1, "}": -1}.get(text[k], 0)
            k += 1
        yield name[1], params, text[j:k]


def test_the_sources_are_understood():
    names = [n for f in FILES for n, _, body in _kernels(_code(f)) if "gridDependencyWait()" in body]
    waits = sum(_code(f).count("gridDependencyWait();") for f in FILES)
    assert {"skipLnKernel", "skipLnQuantKernel", "quantizeRowsKernel", "logProbsKernel", "fcTcgen05PairKernel", "fcTcgen05TileKernel", "fcF32Kernel", "mhaTiledKernel"} <= set(names)
    assert waits >= len(names) > 12


def test_no_parameter_of_such_a_kernel_promises_read_only_data():
    for f in FILES:
        for name, params, body in _kernels(_code(f)):
            if "gridDependencyWait()" in body:
                assert not re.search(r"const\s*\*\s*__restrict__", params), f"{f.name}: {name}"


def test_no_non_coherent_loads_where_such_kernels_are():
    for f in FILES:
        text = _code(f)
        assert "ld.global.nc" not in text, f.name
        kernels = list(_kernels(text))
        plain = [body for _, _, body in kernels if "gridDependencyWait()" not in body]
        if f.suffix == ".cu" and len(plain) == len(kernels):
            continue  # every kernel of the file starts when all before it have ended
        for body in plain:
            text = text.replace(body, "")
        assert "__ldg" not in text, f.name
