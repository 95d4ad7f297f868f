"""bench.py reports the committed counter figures only for the sources they were measured on; the sources left out of
that stamp (kernel_sources_digest) are included by none of the others."""

from __future__ import annotations

import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

APART = {"kv_attn.hip", "kv_cache.hip", "kv_check.h", "kv_layout.h", "qk_rope.hip", "row_types.h", "supra_kv.h"}


def test_measured_kernels_include_none_of_the_sources_left_out():
    for folder in ("supra2-img-web_amd/csrc", "include"):
        for name in os.listdir(os.path.join(ROOT, folder)):
            if name.endswith((".hip", ".h")) and name not in APART:
                with open(os.path.join(ROOT, folder, name)) as f:
                    assert not set(re.findall(r'#include "([^"]+)"', f.read())) & APART, name
