"""The loads to the LDS that the gated layer's kernels issue by hand, in the assembly that the compiler makes of them.  A scalar register that a vector instruction wrote
(a lane read back, for one) may be read by a load five wait states later at the earliest.  The compiler sees to that for its own loads and does not know of these, so that
the distance is looked at here, along every way to each of them."""
import os
import re
import subprocess
import sys

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "..", "arboretum_amd", "csrc")
STATES = 5


def scalars(operand):
    m = re.match(r"s\[(\d+):(\d+)\]$|s(\d+)$|(vcc)", operand)
    if not m:
        return set()
    if m.group(4):
        return {"vcc"}
    return {int(m.group(3))} if m.group(3) else set(range(int(m.group(1)), int(m.group(2)) + 1))


class Kernel:
    """The instructions of a kernel, and where each may come from."""

    def __init__(self):
        self.lines, self.labels = [], {}

    def finish(self):
        self.before = [[] for _ in self.lines]
        for n, words in enumerate(self.lines):
            if words[0].startswith(("s_branch", "s_cbranch")) and words[1] in self.labels and self.labels[words[1]] < len(self.lines):
                self.before[self.labels[words[1]]].append(n)
            if n + 1 < len(self.lines) and words[0] not in ("s_branch", "s_endpgm", "s_setpc_b64"):
                self.before[n + 1].append(n)

    def least(self, load):
        """Wait states from the nearest vector instruction that wrote a scalar register which `load` reads; None where none is within STATES."""
        wanted = frozenset().union(*[scalars(w) for w in self.lines[load][1:]])
        open_ways, seen, found = [(p, wanted, 0) for p in self.before[load]], set(), None
        while open_ways:
            n, wanted, waited = open_ways.pop()
            if waited >= STATES or not wanted or (n, wanted, waited) in seen:
                continue
            seen.add((n, wanted, waited))
            words = self.lines[n]
            written = scalars(words[1]) if len(words) > 1 and not words[0].startswith(("s_cmp", "s_bitcmp", "buffer_store", "global_store")) else set()
            if words[0].startswith("v_") and written & wanted:
                found = waited if found is None else min(found, waited)
                continue
            if words[0].startswith("s_"):
                wanted = wanted - written  # (written by a scalar instruction since: no wait is needed)
            waited += int(words[1], 0) + 1 if words[0] == "s_nop" else 1
            open_ways += [(p, wanted, waited) for p in self.before[n]]
        return found

    def loads(self):
        return [n for n, words in enumerate(self.lines) if words[0].startswith("buffer_load") and "lds" in words]


def kernels(text):
    out, now = {}, None
    for line in text.splitlines():
        line = line.split(";")[0].strip()
        label = re.match(r"^([\w.$]+):", line)
        if label:
            if label.group(1).startswith("_Z"):
                now = out[label.group(1)] = Kernel()
            elif now is not None:
                now.labels[label.group(1)] = len(now.lines)
        elif now is not None and line and not line.startswith("."):
            now.lines.append(line.replace(",", " ").split())
    for kernel in out.values():
        kernel.finish()
    return out


def test_the_reader_of_assembly():
    text = """
_Z1a:
  v_readlane_b32 s4, v1, 0
  s_nop 1
  s_add_u32 m0, s9, 0
  buffer_load_dwordx4 v0, s[4:7], 0 offen lds
.L1:
  buffer_load_dwordx4 v0, s[8:11], 0 offen lds
  s_mov_b32 s4, s5
  s_nop 0
  buffer_load_dwordx4 v0, s[4:7], 0 offen lds
  v_readfirstlane_b32 s8, v2
  s_cbranch_scc1 .L1
  s_endpgm
"""
    kernel = kernels(text)["_Z1a"]
    assert [kernel.least(n) for n in kernel.loads()] == [3, 1, None]


@pytest.mark.parametrize("name", ["gated_bfloat16", "gated_float16", "gated_float32"])
def test_loads_wait_for_what_vector_instructions_wrote(name, tmp_path):
    sys.path.insert(0, os.path.join(HERE, ".."))
    from arboretum_amd.build import FLAGS, hipcc
    out = str(tmp_path / (name + ".s"))
    subprocess.check_call([hipcc()] + FLAGS + ["-Wno-everything", "-x", "hip", "--offload-device-only", "-S", os.path.join(CSRC, name + ".hip"), "-o", out])
    with open(out) as f:
        every = kernels(f.read())
    checked = 0
    for kernel_name, kernel in every.items():
        for load in kernel.loads():
            least = kernel.least(load)
            assert least is None, "%s: %d wait states before %s" % (kernel_name, least, " ".join(kernel.lines[load]))
            checked += 1
    assert checked > 50
