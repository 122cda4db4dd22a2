"""nsparse_amd: MI355X-native hash SpGEMM + AMB SpMV behind the reference's C entry points.

The product is the C-ABI library (include/nsparse.h -> nsparse_amd/lib/libnsparse_{d,s}.so,
sources in nsparse_amd/csrc/).  This Python package only holds the ctypes binding used by the
tests and the bench harness, and the row-sharded multi-GPU driver.

nsparse_amd.lm (include/nsparse_lm.h -> libnsparse_lm.so) has the sparse products of language models on torch tensors;
it imports torch, so it is imported on its own.
"""
from .capi import (load, load_vendor, load_dist, load_lm, Lib, VendorLib, DistLib, LmLib, LmAttn, sfCSR, sfAMB, sfPlan, SpgemmStats,  # noqa: F401
                   SIGNATURES, VENDOR_SIGNATURES, DIST_SIGNATURES, LM_SIGNATURES, DIST_ID_BYTES)
