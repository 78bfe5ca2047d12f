"""Reloads that load nothing, in the kernels that ship (see csrc/sddmm_fused.h: one of them kept a wave in its loop for good).

A divergent loop is left with an empty exec mask: the last lanes took themselves out of it, and the mask of the loop's entry is put back by the first
instruction behind it (s_or_b64 exec, ...).  A vector instruction between the two does nothing.  The compiler has no reason to put one there, but
its register allocator has: a spilled register that is reloaded "behind the loop" and lands in front of the instruction that puts the mask back.
Every kernel that spills, to scratch memory or to accumulation registers, is disassembled and searched for it; no GPU."""
import re
import subprocess

import pytest

from test_isa_cpu import LLVM, kernels  # noqa: F401  (the fixture)


def parse(text):
    """[(address, mnemonic, operands, target address | None)] of one function's disassembly."""
    out, base = [], None
    for line in text.splitlines():
        m = re.match(r'^([0-9a-f]{8,}) <', line)
        if m:
            base = int(m.group(1), 16)
            continue
        m = re.match(r'^\s+(\S+)\s*([^/]*?)\s*// ([0-9A-Fa-f]{8,}):', line)
        if m:
            t = re.search(r'<[^>+]*(?:\+0x([0-9a-f]+))?>\s*$', line)
            out.append((int(m.group(3), 16), m.group(1), m.group(2), base + int(t.group(1) or '0', 16) if t else None))
    return out


def writes_exec(op, args):
    return 'saveexec' in op or (op.startswith('s_') and not op.startswith('s_cbranch') and re.match(r'exec\b', args) is not None)


def empty_reloads(code):
    """Loads from scratch in code that is reached with an empty exec mask only to have it put back: behind a divergent loop, or where a branch on
    the empty mask leads."""
    index = {c[0]: i for i, c in enumerate(code)}
    starts = set()
    for i, (_, op, args, target) in enumerate(code):
        # (a branch on a mask that nothing has narrowed just before is never taken: the compiler's way to fall through)
        if op == 's_cbranch_execz' and target in index and any(writes_exec(c[1], c[2]) for c in code[max(i - 2, 0):i]):
            starts.add(index[target])
        if op == 's_cbranch_execnz' and i and code[i - 1][1] == 's_andn2_b64' and code[i - 1][2].startswith('exec'):
            starts.add(i + 1)
    found = []
    for i in starts:
        for at, op, args, _ in code[i:]:
            if writes_exec(op, args) or op.startswith(('s_cbranch', 's_branch', 's_endpgm', 's_setpc')):
                break
            if op.startswith(('scratch_load', 'v_accvgpr_read')):
                found.append(f'{at:x}: {op} {args}')
    return found


LOOP = """
0000000000001000 <k>:
	s_and_saveexec_b64 s[54:55], vcc                           // 000000001000: BEB6206A
	s_cbranch_execz 6                                          // 000000001004: BF880006 <k+0x20>
	v_add_u32_e32 v7, 64, v7                                   // 000000001008: 680E0EC0
	s_or_b64 s[28:29], vcc, s[28:29]                           // 00000000100C: 879C1C6A
	s_andn2_b64 exec, exec, s[28:29]                           // 000000001010: 89FE1C7E
	s_cbranch_execnz 65531                                     // 000000001014: BF89FFFB <k+0x8>
{behind}
	s_or_b64 exec, exec, s[54:55]                              // 000000001020: 87FE367E
	v_cmp_ge_i32_e32 vcc, s43, v12                             // 000000001024: 7D8C182B
	s_endpgm                                                   // 000000001028: BF810000
"""


def test_the_search_finds_the_reload_and_nothing_else():
    reload_ = '	scratch_load_dword v12, off, off offset:4                  // 000000001018: DC504004 0C7F0000'
    assert empty_reloads(parse(LOOP.format(behind=reload_))) == ['1018: scratch_load_dword v12, off, off offset:4']
    other = '	s_mov_b64 exec, s[54:55]                                   // 000000001018: BEFE0136\n' + reload_.replace('1018', '101C')
    assert empty_reloads(parse(LOOP.format(behind=other))) == []
    assert empty_reloads(parse(LOOP.format(behind=''))) == []


def test_no_kernel_reloads_a_register_for_no_lane(kernels):  # noqa: F811
    by_object = {}
    for co in sorted({k['co'] for k in kernels.values()}):
        notes = subprocess.run([f'{LLVM}/llvm-readelf', '--notes', co], capture_output=True, text=True, check=True).stdout
        for k in re.split(r'\n\s+- \.agpr_count:', notes)[1:]:
            name = re.search(r'\.name:\s+(\S+)', k).group(1)
            if int(re.match(r'\s*(\d+)', k).group(1)) or kernels[name]['scratch']:
                by_object.setdefault(co, []).append(name)
    searched, bad = 0, {}
    for co, names in by_object.items():
        for at in range(0, len(names), 50):
            text = subprocess.run([f'{LLVM}/llvm-objdump', '-d', '--disassemble-symbols=' + ','.join(names[at:at + 50]), co], capture_output=True, text=True, check=True).stdout
            for part in re.split(r'\n(?=[0-9a-f]{16} <)', text):
                m = re.match(r'[0-9a-f]{16} <([^>]+)>:', part)
                if not m:
                    continue
                code = parse(part)
                assert len(code) > 20, m.group(1)
                searched += 1
                found = empty_reloads(code)
                if found:
                    bad[kernels[m.group(1)]['demangled']] = found
    assert searched == sum(len(n) for n in by_object.values()) and searched > 100, searched
    assert not bad, bad
