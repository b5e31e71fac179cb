"""What the compiler checks in its own code and not in inline asm: loads into LDS, which take their
address there from m0, must have the wait states that gfx950 asks for."""
import os
import re
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nanokv-llm_amd", "csrc")
STRING = r'"(?:[^"\\]|\\.)*"'


def _asm_statements():
    """(file, instructions, operands) of every asm statement in csrc, macros put in."""
    read = {f: "\n".join(l for l in open(os.path.join(CSRC, f)).read().split("\n")
                         if not re.match(r"\s*#\s*(include|pragma)", l))
            for f in sorted(os.listdir(CSRC)) if f.endswith((".h", ".hip"))}
    defines = "\n".join(l for t in read.values() for l in t.split("\n") if re.match(r'#define NKV_LDS', l))
    for f, text in read.items():
        text = "\n".join(l for l in text.split("\n") if not re.match(r"\s*#", l))
        text = subprocess.run(["g++", "-E", "-P", "-x", "c++", "-"], input=defines + "\n" + text,
                              capture_output=True, text=True, check=True).stdout
        for m in re.finditer(rf'\basm(?: volatile)?\s*\(((?:[^";]|{STRING})*)\);', text):
            code = re.match(rf"\s*((?:{STRING}\s*)+)", m[1])[1]
            lines = "".join(s[1:-1] for s in re.findall(STRING, code)).replace("\\t", " ").split("\\n")
            yield f, [l.strip() for l in lines if l.strip()], m[1][len(code):]


def test_loads_into_lds_wait_for_m0_and_their_descriptor():
    """One wait state between a write of m0 and the load; five between a vector instruction's write of a
    scalar register and a load whose descriptor it is in. What writes the descriptor stands outside the
    asm, so these five stand in it, counted from its start."""
    found = 0
    for f, lines, operands in _asm_statements():
        states, since_m0 = 0, None
        for l in lines:
            if " m0," in l:
                assert '"m0"' in operands, (f, lines)
                since_m0 = -1  # counted below
            if l.endswith(" lds"):
                found += 1
                assert since_m0 is not None and since_m0 >= 1 and states >= 5, (f, l, lines)
            n = int(l.split()[1]) + 1 if l.startswith("s_nop") else 1
            states += n
            since_m0 = None if since_m0 is None else since_m0 + n
    assert found >= 8  # the statements were read
