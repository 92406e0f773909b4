"""Every entry point that include/lact_b200.h declares is defined within the source's `extern "C"` block: outside of it, a definition whose
parameters have drifted from the declaration compiles as another (C++) function, and the entry is missing without a word."""
import os
import re

from test_abi import ROOT, declared_symbols


def _code(path):
    """The source with comments, texts and characters blanked out (but for the name of the linkage)."""
    s = open(path).read()
    blank = lambda m: '"C"' if m.group(0) == '"C"' else " " * len(m.group(0)) if "\n" not in m.group(0) else "\n" * m.group(0).count("\n")
    return re.sub(r'//[^\n]*|/\*.*?\*/|"(?:\\.|[^"\\\n])*"|\'(?:\\.|[^\'\\\n])+\'', blank, s, flags=re.S)


def test_entry_points_are_defined_within_extern_c():
    s = _code(os.path.join(ROOT, "lact_b200", "csrc", "lact_b200.cu"))
    begin = [m.end() for m in re.finditer(r'extern "C" \{', s)]
    assert len(begin) == 1
    depth, end = 1, begin[0]
    while depth:
        depth += {"{": 1, "}": -1}.get(s[end], 0)
        end += 1
    assert s.count("{") == s.count("}") and not s[end:].strip()          # (the block ends with the file)
    entries = set()
    for m in re.finditer(r"^[a-z][\w *]*[ *](lact_\w+)\(", s, flags=re.M):
        if s[:m.start()].count("{") - s[:m.start()].count("}") == 1 and m.start() > begin[0]:
            entries.add(m.group(1))
    assert entries == set(declared_symbols())
