"""Rules of the machine that the compiler cannot keep for inline assembly, checked in the code it makes."""

import re
import subprocess

import pytest

from reelcache_amd.csrc import build as hip_build

# Vector instructions that write scalar registers, and memory instructions that read them as a resource.
_WRITES = re.compile(r"v_(?:readfirstlane|readlane|cmp)\w* (s\d+|s\[\d+:\d+\])")
_READS = re.compile(r"buffer_(?:load|store|atomic)\w* .*?(s\[\d+:\d+\])")
_WAIT_STATES = 5


def _registers(text):
    first, _, last = text.strip("s[]").partition(":")
    return set(range(int(first), int(last or first) + 1))


def late_resources(assembly):
    """(writer, reader) pairs with fewer than five wait states between a vector write of a scalar register and
    the memory instruction that takes it in its resource."""
    found, window = [], []  # the instructions just before, with the wait states of each
    for line in assembly.splitlines():
        text = line.split(";")[0].strip()
        if not text or text.startswith(".") or text.endswith(":"):
            continue
        if re.match(r"s_branch|s_endpgm|s_setpc", text):  # what follows is entered from elsewhere
            window = []
            continue
        read = _READS.match(text)
        if read:
            wanted, states = _registers(read.group(1)), 0
            for before, worth in reversed(window):
                if states >= _WAIT_STATES:
                    break
                wrote = _WRITES.match(before)
                if wrote and _registers(wrote.group(1)) & wanted:
                    found.append((before, text))
                states += worth
        idle = re.match(r"s_nop (\d+)", text)
        window = window[-_WAIT_STATES:] + [(text, int(idle.group(1)) + 1 if idle else 1)]
    return found


def test_the_check_finds_a_late_resource():
    late = "v_readfirstlane_b32 s44, v32\ns_mov_b32 m0, s1\ns_nop {}\nbuffer_load_dwordx4 v1, s[44:47], 0 offen lds"
    assert len(late_resources(late.format(0))) == 1 and late_resources(late.format(3)) == []
    assert late_resources(late.format(0).replace("s44,", "s48,")) == []


@pytest.mark.parametrize("source", ["attend_rows.hip"])
def test_resources_are_written_early_enough(source, tmp_path):
    """Every assembly block that fetches through a buffer resource waits for the resource's registers."""
    target = tmp_path / "kernels.s"
    subprocess.run([hip_build._hipcc(), *hip_build.FLAGS, "-w", "--cuda-device-only", "-S", str(hip_build.HERE / source), "-o",
                    str(target)], check=True, capture_output=True)
    text = target.read_text()
    assert text.count("offen lds") > 100  # the blocks are in it
    assert late_resources(text) == []
