"""Inline assembly of the kernels names what it writes beside its outputs."""
import re
from pathlib import Path

CSRC = Path(__file__).resolve().parents[1] / "drama3-studio_amd" / "csrc"


def statements():
    for path in sorted(CSRC.glob("*.h*")):
        for m in re.finditer(r"asm\s+volatile\s*\((.*?)\)\s*;", path.read_text(), re.S):
            yield path.name, m.group(1)


def test_m0_is_named_where_it_is_written():
    writing = [(name, text) for name, text in statements() if re.search(r"\bs_\w+\s+m0\s*,", text)]
    assert writing
    for name, text in writing:
        assert '"m0"' in text.rsplit(":", 1)[1], f"{name}: {text}"


def test_barriers_and_waits_order_memory():
    for name, text in statements():
        if re.search(r"\bs_barrier\b|\bs_waitcnt\b", text):
            assert '"memory"' in text.rsplit(":", 1)[1], f"{name}: {text}"
