"""Wait states of the direct-to-LDS loads that inline asm issues, read from the compiler's assembly (no GPU).

The compiler keeps an instruction's wait states for its own instructions, not for inline asm: a load needs one after a
write of m0, and five after a vector instruction that wrote its scalar base (or m0)."""

import re
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

import pytest

PKG = Path(__file__).resolve().parents[1] / "taomate-hd_amd"
SOURCES = ("tmhd_attn", "tmhd_w8a8", "tmhd_mxfp4")


def _scalars(operand):
    """The scalar registers an operand names, by number, and m0."""
    if operand.strip() == "m0":
        return {"m0"}
    found = re.fullmatch(r"s(?:(\d+)|\[(\d+):(\d+)\])", operand.strip())
    if not found:
        return set()
    return set(range(int(found[1] or found[2]), int(found[1] or found[3]) + 1))


def findings(assembly):
    """(loads, those that come too early): each load's line and what it comes too early behind."""
    loads, early, before = 0, [], []  # before: (wait states it gives, opcode, scalars written)
    for line in assembly.splitlines():
        text = line.split(";")[0].strip()
        if text.endswith(":") and not text.startswith("."):
            before = []  # a function's first instruction
        if not text or text.startswith((".", "#")) or text.endswith(":"):
            continue
        op, _, rest = text.partition(" ")
        operands = rest.split(",")
        if op.startswith("global_load_lds"):
            loads += 1
            base, states = _scalars(operands[1].split()[0]), 0
            for waits, by, written in reversed(before):
                needs = 5 if by.startswith("v_") else 1
                if (written & (base | {"m0"}) if needs == 5 else "m0" in written) and states < needs:
                    early.append(f"{text} behind {by}")
                states += waits
                if states >= 5:
                    break
        waits = int(operands[0], 0) + 1 if op == "s_nop" else 1
        before = [*before[-5:], (waits, op, _scalars(operands[0]) if op[:2] in ("s_", "v_") else set())]
    return loads, early


def test_findings_of_short_listings():
    load = "global_load_lds_dwordx4 v1, s[4:5]\n"
    assert findings("f:\ns_mov_b32 m0, s1\n" + load) == (1, ["global_load_lds_dwordx4 v1, s[4:5] behind s_mov_b32"])
    assert findings("f:\ns_mov_b32 m0, s1\ns_nop 0\n" + load) == (1, [])
    assert len(findings("f:\nv_readlane_b32 s5, v9, 3\ns_nop 3\n" + load)[1]) == 1
    assert findings("f:\nv_readlane_b32 s5, v9, 3\ns_nop 4\n" + load) == (1, [])
    assert findings("f:\nv_readlane_b32 s6, v9, 3\n" + load) == (1, [])
    assert findings("f:\nv_readlane_b32 s6, v9, 3\ns_mov_b64 s[4:5], s[6:7]\n" + load) == (1, [])
    assert findings("f:\ns_mov_b32 s5, 0\n" + load) == (1, [])


@pytest.fixture(scope="module")
def listings(tmp_path_factory):
    sys.path.insert(0, str(PKG))
    try:
        import build
    finally:
        sys.path.remove(str(PKG))
    out = tmp_path_factory.mktemp("listings")
    flags = [f for f in build.HIPCC_FLAGS if f not in ("-fPIC", "-Wall")]

    def listing(name):
        cmd = [build._hipcc(), *flags, "-S", "--offload-device-only", str(PKG / "csrc" / f"{name}.hip"), "-o", str(out / f"{name}.s")]
        run = subprocess.run(cmd, capture_output=True, text=True, timeout=600)
        assert run.returncode == 0, run.stderr[-2000:]
        return (out / f"{name}.s").read_text()

    with ThreadPoolExecutor(len(SOURCES)) as pool:
        return dict(zip(SOURCES, pool.map(listing, SOURCES)))


@pytest.mark.parametrize("source", SOURCES)
def test_loads_keep_their_wait_states(listings, source):
    loads, early = findings(listings[source])
    assert loads > 50
    assert not early, (len(early), early[:5])
