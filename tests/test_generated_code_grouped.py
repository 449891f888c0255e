"""The checks of test_generated_code.py on the grouped products' source (CPU only: cross-compiles to assembly): its
big-tile kernel issues the same direct loads and in-place matrix instructions from inline assembly."""
import re
import subprocess

import pytest

import test_generated_code as gen
from prism_amd import build as pbuild

SOURCE = "gemm_grouped.hip"


@pytest.fixture(scope="module")
def text(tmp_path_factory):
    out = tmp_path_factory.mktemp("asm") / (SOURCE + ".s")
    cmd = [pbuild.hipcc_path(), *pbuild.HIPCC_FLAGS, "-S", "--cuda-device-only", "-o", str(out), str(pbuild.CSRC / SOURCE)]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    assert proc.returncode == 0, proc.stderr[-2000:]
    return out.read_text()


def test_direct_loads(text):
    gen.test_every_direct_load_has_its_own_m0_write({SOURCE: text}, SOURCE)
    gen.test_no_vector_written_scalar_is_read_by_a_direct_load_too_soon({SOURCE: text}, SOURCE)
    assert not re.search(r"buffer_load_dwordx4 v\d+, v\[", text), "a descriptor in vector registers"


def test_matrix_instructions(text):
    """The accumulator check goes by its kernel's name: the grouped kernels are shown to it under that name."""
    shown = {"gemm_bf16.hip": re.sub(r"gemm_grouped(_big)?_kernel", "gemm_bf16_early_kernel", text)}
    gen.test_no_matrix_instruction_reads_a_register_the_vector_alu_has_just_written(shown)
    gen.test_no_accumulator_is_read_too_soon_after_an_in_place_matrix_instruction(shown)


def test_no_spills_and_nothing_but_the_pipeline_in_the_k_loop(text):
    kernels = re.findall(r"^\s*\.amdhsa_kernel\s+(\S*gemm_grouped_big_kernel\S*)(.*?)\.end_amdhsa_kernel", text, re.S | re.M)
    assert len(kernels) == 6
    for name, body in kernels:
        assert re.search(r"\.amdhsa_private_segment_fixed_size\s+0\b", body), name
    # the K loops (the only loops of 256 matrix instructions): no accumulator moves, at most two vector instructions a phase and operand
    found, lines, labels, kernel = 0, [], {}, None
    for raw in text.splitlines():
        line = raw.split(";")[0].strip()
        if line.startswith("_Z") and line.endswith(":"):
            kernel, lines, labels = line, [], {}
            continue
        if kernel is None or "gemm_grouped_big_kernel" not in kernel or not line:
            continue
        if line.startswith(".LBB"):
            labels[line[:-1]] = len(lines)
        lines.append(line)
        branch = re.match(r"s_cbranch\w*\s+(\.LBB\S+)", line)
        if branch and branch.group(1) in labels:
            loop = lines[labels[branch.group(1)]:]
            if sum(i.startswith("v_mfma") for i in loop) == 256:
                found += 1
                assert not any(i.startswith(("v_accvgpr", "scratch_")) for i in loop), kernel
                assert sum(i.startswith("v_") and not i.startswith(("v_mfma", "v_readlane")) for i in loop) <= 8, kernel
    assert found >= 6
