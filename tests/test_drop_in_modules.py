"""`install_as_triton_kernels()`: a module has one copy, whichever of the two names it is imported by."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PACKAGE = os.path.join(ROOT, "triton_amd")


def public_modules():
    for folder, folders, files in os.walk(PACKAGE):
        folders[:] = [d for d in folders if not d.startswith("_") and os.path.exists(os.path.join(folder, d, "__init__.py"))]
        at = os.path.relpath(folder, PACKAGE).replace(os.sep, ".")
        for f in files:
            if f.endswith(".py") and not f.startswith("_") and f != "build.py":   # (build.py is a command)
                yield f[:-3] if at == "." else f"{at}.{f[:-3]}"
        for d in folders:
            yield d if at == "." else f"{at}.{d}"


def test_the_list_is_whole():
    assert {"matvec", "moe_layer", "sampling", "matmul", "tensor_details.layout", "numerics_details.mxfp"} <= set(public_modules())


def test_one_copy():
    """(In a process of its own: what another test has imported would hide a second copy.)"""
    code = ("import triton_amd, importlib, sys; triton_amd.install_as_triton_kernels()\n"
            "two = [n for n in sys.argv[1:] if importlib.import_module('triton_kernels.' + n) is not importlib.import_module('triton_amd.' + n)]\n"
            "assert not two, two")
    subprocess.run([sys.executable, "-c", code, *sorted(public_modules())], cwd=ROOT, check=True, timeout=100)


def test_packed_weights_have_one_class():
    code = ("import triton_amd; triton_amd.install_as_triton_kernels()\n"
            "from triton_kernels.matvec import Int4Weights, matvec\nimport triton_amd.matvec as own\n"
            "assert Int4Weights is own.Int4Weights and matvec is own.matvec")
    subprocess.run([sys.executable, "-c", code], cwd=ROOT, check=True, timeout=100)
