"""The library holds no kernel of the operators on microscaled rows that no call reaches."""
import re

import pytest


def kernels(hip):
    """The instances of gemm_mx_* and rms_norm_* kernels among the library's names: {kernel: {template arguments as mangled}}."""
    found = {}
    with open(hip.LIB_PATH, "rb") as f:
        for name, args in set(re.findall(rb"\d+(gemm_mx_[a-z]+_kernel|rms_norm[a-z_]*_kernel)I(\w+?)EEv", f.read())):
            found.setdefault(name.decode(), set()).add(args.decode())
    return found


@pytest.mark.parametrize("kernel,never", [
    ("gemm_mx_stream_kernel", "Lb1Ef"), ("gemm_mx_tile_kernel", "Lb1Ef"),          # 8-bit rows to float32 are refused
    ("rms_norm_kernel", "fLi64ELi3"), ("rms_norm_kernel", "fLi256ELi3"),            # float32 rows gain nothing from three loads to a thread
    ("rms_norm_kernel", "fLi512ELi4"), ("rms_norm_backward_kernel", "fLi512ELi4"),  # float32 rows past 12288 values: 1024 threads
    ("rms_norm_kernel", "Bf16ELi1024E"), ("rms_norm_kernel", "DF16_Li1024E"),       # 16-bit ones: 512
    ("rms_norm_backward_kernel", "Bf16ELi1024E"), ("rms_norm_backward_kernel", "DF16_Li1024E"),
    ("rms_norm_backward_kernel", "Li256ELi3")])                                    # the gradient loses by it
def test_no_kernel_that_no_call_reaches(hip, kernel, never):
    found = kernels(hip)
    assert len(found["gemm_mx_stream_kernel"]) >= 30 and len(found["rms_norm_kernel"]) >= 20        # (they are seen at all)
    assert not [args for args in found[kernel] if never in args]
