"""The copies of cross_attention.hip that write LDS without passing registers: compiled by the builtin, and by the
intrinsic's name as for a compiler that lacks the builtin. The instructions are the same."""
import os
import re
import subprocess

import pytest

from devspace_amd.ops import build

ABSENT = "!__has_builtin(__builtin_amdgcn_raw_ptr_buffer_load_lds)"
AROUND = """#include <hip/hip_runtime.h>
typedef __attribute__((address_space(3))) unsigned char lds_u8;
typedef __attribute__((address_space(3))) void lds_void;
%s
extern "C" __global__ void probe(const char* from, unsigned bytes, float4* to) {
  __shared__ __attribute__((aligned(16))) float4 wide[64];
  __shared__ float narrow[64];
  to_lds<16>(from, bytes, wide, threadIdx.x * 16);
  to_lds<4>(from, bytes, narrow, threadIdx.x * 4);
  __syncthreads();
  to[threadIdx.x] = wide[63 - threadIdx.x];
  to[threadIdx.x].x += narrow[63 - threadIdx.x];
}
"""


def _instructions(text, at):
    src, out = at + ".hip", at + ".s"
    with open(src, "w") as f:
        f.write(AROUND % text)
    subprocess.run([build.hipcc(), "-O3", f"--offload-arch={build.ARCH}", *build.NO_PACKED_FP32, "-std=c++17", "-S",
                    "--cuda-device-only", "-o", out, src], check=True, timeout=300, stderr=subprocess.DEVNULL)
    with open(out) as f:
        body = f.read()
    body = body[body.index("probe:"):body.index("s_endpgm")]
    return [" ".join(line.split(";")[0].split()) for line in body.split("\n") if re.match(r"\s+[a-z]", line)]


def test_both_forms_are_the_same_instructions(tmp_path):
    try:
        build.hipcc()
    except FileNotFoundError:
        pytest.skip("needs hipcc")
    with open(os.path.join(build.HERE, "cross_attention.hip")) as f:
        source = f.read()
    part = source[source.rindex("#if", 0, source.index(ABSENT)):source.index("// N chunks of 16 bytes")]
    here = _instructions(part, str(tmp_path / "here"))
    named = _instructions(part.replace(ABSENT, "1"), str(tmp_path / "named"))
    assert here == named
    loads = [i for i in here if i.startswith("buffer_load") and i.endswith(" lds")]
    assert [i.split()[0] for i in loads] == ["buffer_load_dwordx4", "buffer_load_dword"]
