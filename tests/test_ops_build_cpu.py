"""What the model operators' device helpers compile to: checked on the assembly that hipcc writes, without a GPU."""

import os
import re
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tandem_amd", "csrc")


def test_every_offset_of_a_buffer_access_is_compared_with_its_end(tmp_path):
    """load16 / store16 reach behind a row's end on purpose: the hardware's comparison keeps them out. The scalar offset of a raw buffer
    instruction is not promised to take part in it, so it has to be zero, also where a constant does not fit the instruction."""
    from tandem_amd.build import FLAGS

    source = tmp_path / "stretch.hip"
    source.write_text(f'''#include "{CSRC}/ops_device.h"
using namespace tandem_hip::ops;
extern "C" __global__ void copy(const void* from, void* to, int bytes) {{
  const auto a = stretch(from, bytes), b = stretch(to, bytes);
#pragma unroll
  for (int i = 0; i < 4; ++i) store16(load16(a, threadIdx.x * 16, i * 16384), b, threadIdx.x * 16, i * 16384);
}}
''')
    out = tmp_path / "stretch.s"
    subprocess.run([os.environ.get("HIPCC", "/opt/rocm/bin/hipcc"), *FLAGS, "-w", "--offload-device-only", "-S", str(source), "-o", str(out)], check=True)
    accesses = re.findall(r"buffer_(?:load|store)_dwordx4 \S+ \S+ s\[\d+:\d+\], (\S+)", out.read_text())
    assert len(accesses) == 8 and set(accesses) == {"0"}, accesses
