"""Loads into LDS that are written as inline assembly keep the wait states the compiler does not insert for them: compiled for gfx950
here, their assembly is looked at."""
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SOURCE = """
#include "lds_dma.h"
__global__ void k_bounded(const uint64_t *base, const uint32_t *records, const uint32_t *off) {
  __shared__ __attribute__((aligned(1024))) unsigned char ring[1024];
  const anc_i32x4 b = buffer_of((const char *)base[threadIdx.x], records[threadIdx.x]);
  dma16_bounded(b, off[threadIdx.x], lds_addr(ring));
  wait_vm<0>();
}
__global__ void k_uniform(const uint64_t *base, const uint32_t *off) {
  __shared__ __attribute__((aligned(1024))) unsigned char ring[1024];
  const uint64_t v = base[threadIdx.x];
  const uint64_t b = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(v >> 32)) << 32 |
                     (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)v);
  dma16((const void *)b, off[threadIdx.x], lds_addr(ring));
  wait_vm<0>();
}
"""


def _registers(text):
    """Scalar registers that an operand list names."""
    out = set()
    for a, b in re.findall(r"\bs\[(\d+):(\d+)\]", text):
        out |= set(range(int(a), int(b) + 1))
    return out | {int(a) for a in re.findall(r"\bs(\d+)\b", text)}


def _shortest_wait(body):
    """Fewest wait states between a vector instruction's write of a scalar register and a load into LDS that reads it."""
    written, now, short = {}, 0, []
    for line in body:
        op, _, args = line.strip().partition(" ")
        if re.match(r"(global|buffer)_load_(lds_)?dwordx4", op) and ("lds" in line):
            short += [now - written[r] for r in _registers(args) if r in written]
        elif op.startswith("v_"):
            to = args.split(",")[0]
            for r in _registers(to):
                written[r] = now + 1
        elif op.startswith("s_") and not op.startswith(("s_nop", "s_waitcnt", "s_cmp")):
            for r in _registers(args.split(",")[0]):
                written.pop(r, None)                    # (a scalar write is waited for by the hardware)
        now += 1 + (int(args) if op == "s_nop" else 0)
    return min(short) if short else None


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    from ancora_cutile_amd import build
    at = tmp_path_factory.mktemp("isa")
    (at / "probe.hip").write_text(SOURCE)
    subprocess.run([os.environ.get("HIPCC", "/opt/rocm/bin/hipcc"), *[f for f in build.FLAGS if f not in ("-shared", "-fPIC")], "-S", "--cuda-device-only",
                    "-I", build.CSRC, "-I", os.path.join(ROOT, "include"), str(at / "probe.hip"), "-o", str(at / "probe.s")], check=True, capture_output=True, timeout=300)
    found, name = {}, None
    for line in (at / "probe.s").read_text().split("\n"):
        m = re.match(r"_Z\d+(k_\w+?)P", line)
        if m and line.split(";")[0].strip().endswith(":"):
            name = m.group(1)
            found[name] = []
        elif name and re.match(r"\s+[a-z]", line) and not line.strip().startswith("."):
            found[name].append(line.split(";")[0])
        if name and "s_endpgm" in line:
            name = None
    return found


@pytest.mark.parametrize("kernel,waits", [("k_bounded", True), ("k_uniform", False)])
def test_a_scalar_register_that_a_vector_instruction_wrote_is_waited_for(kernels, kernel, waits):
    body = kernels[kernel]
    assert any("v_readfirstlane" in line for line in body) and any("lds" in line for line in body)
    wait = _shortest_wait(body)
    if waits:
        assert wait is not None and wait >= 5, body
    else:
        assert wait is None, body                       # copied by a scalar instruction first
