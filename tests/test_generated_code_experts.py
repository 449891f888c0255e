"""Checks of what the compiler makes of the expert-layer kernels (CPU only: cross-compiles to assembly)."""
import re

from test_generated_code_grouped import text  # noqa: F401 (the grouped products' assembly)


def kernel_bodies(text, pattern):  # noqa: F811
    """{name: instruction lines and labels} of the kernels whose mangled name matches."""
    out, name = {}, None
    for raw in text.splitlines():
        line = raw.split(";")[0].strip()
        if line.startswith("_Z") and line.endswith(":"):
            name = line[:-1] if re.search(pattern, line) else None
            if name:
                out[name] = []
        elif line.startswith(".section") or line.startswith(".amdhsa_kernel"):
            name = None
        elif name and line and (not line.startswith(".") or line.startswith(".LBB")):
            out[name].append(line)
    return out


def test_a_stage_by_ordinary_loads_ends_with_a_wait_for_all_loads(text):  # noqa: F811
    """The barriers of the four-stage ring count on eight direct loads a stage. A wavefront can be without any ordinary load
    in a stage that comes by ordinary loads, so behind the writes of its packets (ds_write_b128) stands a wait for every load,
    on the way to the next direct load, barrier or read, whatever the waits in front of the writes cover."""
    kernels = kernel_bodies(text, r"gemm_grouped_kernelILb[01]ELb[01]ELb[01]ELb0ELi4E")
    assert len(kernels) == 6
    for name, lines in kernels.items():
        at = {line[:-1]: i for i, line in enumerate(lines) if line.startswith(".LBB")}
        writes = [i for i, line in enumerate(lines) if line.startswith("ds_write_b128")]
        assert len(writes) >= 8, name
        ends = 0
        for i in writes:
            i += 1
            while True:
                line = lines[i]
                if re.match(r"s_waitcnt\b.*\bvmcnt\(0\)", line):
                    ends += 1
                    break
                if line.startswith(("ds_write_b128", "global_load")):  # the stage's next packet
                    break
                assert not re.match(r"buffer_load|s_barrier|ds_read|s_endpgm", line), f"{name}: {line}"
                i = at[line.split()[1]] if line.startswith("s_branch") else i + 1
        assert ends >= 4, name  # three stages ahead of the loop, and the one in it
