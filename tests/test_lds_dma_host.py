"""Host: the asm statements that load straight into LDS keep the wait state between the write of m0 and the load."""
import glob
import os
import re

CSRC = os.path.join(os.path.dirname(__file__), "..", "obman_train_amd", "csrc")


def _statements(source):
    """The instruction lists of the source's asm statements (adjacent literals joined)."""
    for m in re.finditer(r"\basm\s+(?:volatile\s*)?\(\s*((?:\"(?:[^\"\\]|\\.)*\"\s*)+)", source):
        text = "".join(re.findall(r"\"((?:[^\"\\]|\\.)*)\"", m.group(1)))
        yield [i.strip() for i in re.split(r"\\n(?:\\t)?|;", text) if i.strip()]


def _without_wait(instructions):
    return [b for a, b in zip(instructions, instructions[1:]) if re.match(r"s_\w+ m0\b", a) and re.search(r"\blds\b", b)]


def test_the_check_sees_what_it_is_for():
    bad, = _statements('asm volatile("s_mov_b32 m0, %0\\n\\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(a));')
    good, = _statements('asm volatile("s_mov_b32 m0, %0\\n\\ts_nop 0\\n\\t"\n "buffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(a));')
    assert _without_wait(bad) and not _without_wait(good)


def test_a_load_to_lds_is_not_the_instruction_behind_the_write_of_m0():
    loads = 0
    for path in sorted(glob.glob(os.path.join(CSRC, "*.h*"))):
        with open(path) as f:
            for instructions in _statements(f.read()):
                loads += any(re.search(r"\blds\b", i) for i in instructions)
                assert not _without_wait(instructions), (os.path.basename(path), instructions)
    assert loads >= 2
