"""Finds divergent blocks of compiled gfx950 code that do nothing: exec narrowed by s_and_saveexec_b64 and
restored right behind it. The source asked for something there, so the compiler has dropped it.

It does that to `if (!there || a > b || a <= c) x = -inf;` where `there` is one for the wave and the others are a
lane's: of several such statements in a row the last one's move stays in the block of the uniform condition alone,
and lanes that the others pick keep their x."""
import re


def empty_blocks(asm):
    """(kernel, line) of every such block in assembly as hipcc -S writes it."""
    kernel, narrowed, found = None, None, []
    for number, line in enumerate(asm.splitlines(), 1):
        label = re.match(r"(_Z\S+):", line)
        if label:
            kernel, narrowed = label.group(1), None
            continue
        code = line.split(";")[0].strip()
        if not code or code.startswith("."):
            continue
        if code.startswith("s_and_saveexec_b64"):
            narrowed = (number, code.split()[1].rstrip(","))
        elif narrowed:
            if code == f"s_or_b64 exec, exec, {narrowed[1]}":
                found.append((kernel, narrowed[0]))
            if not code.startswith(("s_waitcnt", "s_nop", "s_cbranch_execz")):
                narrowed = None
    return found
