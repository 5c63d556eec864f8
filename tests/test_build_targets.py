"""What the library's makefile builds by itself, and what it needs for it."""
import os
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "provenloop_amd", "csrc")


def plan(*args):
    return subprocess.run(["make", "-n", "-B", "-C", CSRC, *args], capture_output=True, text=True)


def test_the_library_needs_neither_torch_nor_python():
    p = plan("PYTHON=/no/such/python")
    assert p.returncode == 0 and "libtensafe_he_hip.so" in p.stdout
    assert "torch" not in p.stdout and "/no/such/python" not in p.stdout + p.stderr


def test_the_binding_is_a_target_of_its_own():
    p = plan("mixture")
    assert p.returncode == 0 and "-ltorch_hip" in p.stdout and "_mixture_torch.so" in p.stdout
