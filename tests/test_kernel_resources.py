"""CPU: what the compiler gave the kernels of the built library, read from the metadata of its gfx950 code objects (compiled from this tree's sources)."""
import os
import re
import struct
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(ROOT, "fastllama_amd", "libfastllama_hip.so")
READELF, OBJDUMP = (os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "llvm", "bin", x) for x in ("llvm-readelf", "llvm-objdump"))


def code_objects(data):
    """The ELF images for AMD GPUs (machine 224) inside the library, from header to the end of their section table."""
    at = data.find(b"\x7fELF", 1)
    while at >= 0:
        if struct.unpack_from("<H", data, at + 18)[0] == 224:
            table, = struct.unpack_from("<Q", data, at + 40)
            size, count = struct.unpack_from("<HH", data, at + 58)
            yield data[at:at + table + size * count]
        at = data.find(b"\x7fELF", at + 4)


@pytest.fixture(scope="module")
def scratch(tmp_path_factory):
    """{demangled kernel: bytes of scratch a lane}"""
    if not os.path.exists(READELF):
        pytest.skip("llvm-readelf is not installed")
    if not os.path.exists(LIB):
        subprocess.check_call([os.path.join(ROOT, "build.sh")])
    found, file = {}, tmp_path_factory.mktemp("code") / "object"
    for image in code_objects(open(LIB, "rb").read()):
        file.write_bytes(image)
        notes = subprocess.run([READELF, "--notes", str(file)], capture_output=True, text=True, check=True).stdout
        for kernel in re.split(r"^  - ", notes.split("amdhsa.kernels:")[-1], flags=re.M)[1:]:
            name, size = re.search(r"\.name:\s+(\S+)", re.sub(r"^ {8,}.*\n", "", kernel, flags=re.M)), re.search(r"\.private_segment_fixed_size:\s+(\d+)", kernel)
            if name and size:
                found[name.group(1)] = int(size.group(1))
    names = subprocess.run(["c++filt"], input="\n".join(found), capture_output=True, text=True, check=True).stdout.split("\n")
    return dict(zip(names, found.values()))


def test_streaming_decode_kernels_keep_their_registers(scratch):
    """The one-wave-per-row-group kernel of a decode step has its weights in flight in registers: one that spills waits for scratch memory in its loop."""
    kernels = {k: v for k, v in scratch.items() if "gemv1_q4_exact_stream_kernel" in k}
    assert len(kernels) >= 30
    assert not {k: v for k, v in kernels.items() if v}


def loops(lines):
    """The bodies of a kernel's loops: [(address, instruction)] from a backward branch's target to the branch."""
    at = {a: i for i, (a, _) in enumerate(lines)}
    for i, (a, text) in enumerate(lines):
        m = re.match(r"s_c?branch\S*\s+(\d+)", text)
        if m and int(m.group(1)) > 32767:                     # words back from the next instruction
            first = at.get(a + 4 + 4 * (int(m.group(1)) - 65536))
            if first is not None:
                yield lines[first:i + 1]


def test_streaming_decode_loops_do_not_wait_for_all_their_loads(scratch, tmp_path):
    """The norm forms of the one-wave-per-row-group kernel keep 8 or 16 quads of weights on their way: nowhere in the loop may they wait for the last of them."""
    if not os.path.exists(OBJDUMP):
        pytest.skip("llvm-objdump is not installed")
    seen, waits = 0, {}
    for image in code_objects(open(LIB, "rb").read()):
        if b"gemv1_q4_exact_stream_kernel" not in image:
            continue
        (tmp_path / "object").write_bytes(image)
        text = subprocess.run([OBJDUMP, "-d", "--demangle", str(tmp_path / "object")], capture_output=True, text=True, check=True).stdout
        for name, body in re.findall(r"^[0-9a-f]+ <(.*)>:\n((?:\t.*\n)+)", text, flags=re.M):
            if not re.search(r"gemv1_q4_exact_stream_kernel<[23], 1, ", name):
                continue
            lines = [(int(a, 16), t) for t, a in re.findall(r"^\t(.*?)\s*// ([0-9A-F]+):", body, flags=re.M)]
            for loop in loops(lines):
                if sum("buffer_load_dwordx4" in t for _, t in loop) in (8, 16):
                    seen += 1
                    least = min(int(m.group(1)) for _, t in loop for m in [re.search(r"vmcnt\((\d+)\)", t)] if m)
                    if least < 8:
                        waits[name] = least
    assert seen >= 30 and not waits


@pytest.mark.parametrize("kernel", ["attn_prompt_k", "attn_prompt_join_k", "attn_decode_k", "attn_join_k", "kv_append_k", "sample_scan_k", "sample_hist_k", "sample_gather_k",
                                    "sample_draw_k"])
def test_operators_over_several_sequences_use_no_scratch(scratch, kernel):
    """Their entry points allocate nothing, so no launch of theirs may make the runtime allocate scratch memory."""
    kernels = {k: v for k, v in scratch.items() if kernel in k}
    assert len(kernels) >= 3
    assert not {k: v for k, v in kernels.items() if v}
