"""What compiled assembly has to hold that neither the compiler nor a run shows reliably."""

import os
import re
import subprocess

from libcertex_amd import build

PROBE = """#include <attention/tiles.hpp>
using namespace certex_amd::attention;
__global__ void copies(const char* const* from, const int* slots, float* to)
{
  __shared__ __attribute__((aligned(16))) float s[2][256];
  const char* base = from[threadIdx.x];  // of lane 0, read by a vector instruction
  copy_to_lds(base, threadIdx.x * 16, uniform(slots[threadIdx.x]));
  copy_to_lds(base + threadIdx.x * 4, lds_address(s[1]));
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  to[threadIdx.x] = s[0][threadIdx.x] + s[1][threadIdx.x];
}
"""


def compiled(tmp_path, text, *how):
    """The assembly of a source (or what `how` asks for instead), and what the compiler said."""
    path, out = tmp_path / "probe.hip", tmp_path / "probe.s"
    path.write_text(text)
    cmd = [build.HIPCC, "-x", "hip", *build.COMMON, "-I", build.CSRC, "--cuda-device-only", "-S", str(path), "-o", str(out), *how]
    r = subprocess.run(cmd, capture_output=True, text=True)
    return out.read_text() if r.returncode == 0 else None, r.stderr


def scalars(operand):
    """The scalar registers of an operand."""
    many, one = re.match(r"s\[(\d+):(\d+)\]", operand), re.match(r"s(\d+)\b", operand)
    return set(range(int(many[1]), int(many[2]) + 1)) if many else {int(one[1])} if one else {operand}


def wait_states(assembly):
    """Per copy to LDS: the wait states since a lane read wrote one of the scalar registers that it reads, if one did (None)."""
    states, before = [], []
    for line in assembly.splitlines():
        line = line.split(";")[0].strip()
        if not line or line[0] == "." or line.endswith(":"):
            continue
        op, _, rest = line.partition(" ")
        args = [x.strip() for x in rest.split(",")]
        if op.startswith("global_load_lds"):
            reads, passed, found = scalars(args[1].split()[0]) | {"m0"}, 0, None
            for other, writes, n in reversed(before):
                if other.startswith(("v_readfirstlane", "v_readlane")) and scalars(writes) & reads:
                    found = passed
                    break
                passed += n
            states.append(found)
        before.append((op, args[0], int(args[0]) + 1 if op == "s_nop" else 1))
    return states


def test_copies_to_lds_wait_for_their_address(tmp_path):
    """A scalar register that a vector instruction wrote is read by a memory instruction 5 wait states later at the earliest. The
    compiler does not see the copies, which are assembly: they hold the states themselves."""
    assembly, said = compiled(tmp_path, PROBE)
    states = wait_states(assembly)
    assert len(states) == 2 and states[0] is not None, said  # the probe does read lanes for the first copy's address
    assert all(n is None or n >= 5 for n in states), states


def test_copies_to_lds_clobber_no_reserved_register(tmp_path):
    """The copies' register M0 is an operand: named as clobbered, which the compiler only warns of, it would be undefined."""
    assert "-Werror=inline-asm" in build.COMMON
    assembly, said = compiled(tmp_path, PROBE)
    assert assembly and "reserved register" not in said, said
    assembly, said = compiled(tmp_path, PROBE.replace("vmcnt(0)\" ::: ", "vmcnt(0)\" ::: \"m0\", "))
    assert assembly is None and "reserved register" in said


def test_packed_keys_are_aligned_as_promised(tmp_path):
    """csrc/attention/attention.hpp: every piece of a packed key, for all head dimensions, begins where the kernels say."""
    exe = tmp_path / "packed_align"
    source = os.path.join(os.path.dirname(__file__), "c", "packed_align.cpp")
    subprocess.run([build.HIPCC, "-x", "hip", *build.COMMON, "--offload-host-only", "-I", build.CSRC, "-fvisibility=default", source,
                    "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout == "ok\n", r.stdout
