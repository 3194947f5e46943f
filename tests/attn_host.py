"""What attn.hip decides on the host (libosmos_amd/csrc/attnhost.h), compiled by itself for the tests that need no GPU."""
import ctypes
import os
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))


def build(folder):
    lib = os.path.join(str(folder), "attn_host.so")
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", os.path.join(HERE, "attn_host_driver.cpp"),
                    "-o", lib], check=True)
    return ctypes.CDLL(lib)
