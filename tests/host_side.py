"""The library's host side without a GPU: a child process loads fake_hip.cpp's calls before
libbchip.so, which then binds to them, and runs a test's body with

  c            a context
  mallocs()    (address, bytes, serial number) of every hipMalloc since clear()
  launches()   (kernel, its grid) of every launch since clear(); none of them runs
  clear()
  live(m)      whether such a block is still allocated
  capturing()  a `with` during which the stream counts as captured and hipMalloc fails
  refused(code, call)"""
import os
import subprocess
import sys
import textwrap

HERE = os.path.dirname(os.path.abspath(__file__))

PRELUDE = """
import contextlib, ctypes, os, sys
import numpy as np
fake = ctypes.CDLL({fake!r}, mode=ctypes.RTLD_GLOBAL)
sys.path[:0] = {path!r}
import bchip
fake.fake_malloc_at.restype, fake.fake_launch.restype = ctypes.c_void_p, ctypes.c_char_p
fake.fake_malloc_at.argtypes, fake.fake_launch.argtypes = [ctypes.c_size_t, ctypes.c_void_p, ctypes.c_void_p], [ctypes.c_size_t]
fake.fake_live.argtypes, fake.fake_budget.argtypes = [ctypes.c_void_p, ctypes.c_size_t], [ctypes.c_size_t]
def mallocs():
    n, k = ctypes.c_size_t(), ctypes.c_size_t()
    return [(fake.fake_malloc_at(i, ctypes.byref(n), ctypes.byref(k)), n.value, k.value) for i in range(fake.fake_mallocs())]
def launches():
    got = [fake.fake_launch(i).decode().split() for i in range(fake.fake_launches())]
    return [(name, tuple(map(int, grid))) for name, *grid in got]
clear, live = fake.fake_clear, lambda m: fake.fake_live(m[0], m[2])
@contextlib.contextmanager
def capturing():
    fake.fake_capture(1)
    try:
        yield
    finally:
        fake.fake_capture(0)
def refused(code, call):
    clear()
    try:
        call()
    except bchip.BchipError as e:
        assert e.code == code, (e.code, bchip.last_error())
        assert not launches(), launches()
    else:
        raise AssertionError("not refused")
c = bchip.Ctx(0)
"""


def build(to):
    """fake_hip.cpp as a library in the folder `to`."""
    so = os.path.join(str(to), "fake_hip.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-w", "-shared", "-fPIC", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include",
                    os.path.join(HERE, "fake_hip.cpp"), "-o", so], check=True)
    return so


def run(fake, body):
    root = os.path.dirname(HERE)
    path = [os.path.join(root, "borrowed-compute_amd"), os.path.join(root, "oracle"), HERE]
    code = PRELUDE.format(fake=fake, path=path) + textwrap.dedent(body)
    out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0, out.stdout + out.stderr
    return out.stdout
