"""The tile kernels of the 8-bit product issue their matrix instructions where the compiler does not see them, so that it keeps none of the
distances that the hardware asks for between such an instruction and others on its registers.  Here the built code is
followed over all its branches: whatever else reads or writes a matrix instruction's sums comes 19 or more wait states behind it (what the
longest of them needs), unless a matrix instruction has taken them over with the very same sums; and no other vector
instruction writes a register that a matrix instruction reads within the next two."""
import re

from tests.test_native_jumps import kernels

BEHIND, BEFORE = 19, 2


def registers(operand):
    """the vector and accumulation registers of an operand, as ("a", 5)"""
    out = set()
    for kind, one, lo, hi in re.findall(r"(?<![a-z_])([va])(?:(\d+)|\[(\d+):(\d+)\])", operand):
        out |= {(kind, int(one))} if one else {(kind, i) for i in range(int(lo), int(hi) + 1)}
    return out


class Code:
    def __init__(self, code):
        self.code = code
        at = {address: i for i, (address, _, _) in enumerate(code)}
        self.used = [[registers(o) for o in ops] for _, _, ops in code]
        self.touched = [set().union(*u) if u else set() for u in self.used]
        self.next = []
        for i, (address, name, ops) in enumerate(code):
            after = [i + 1] if i + 1 < len(code) else []
            if name.startswith(("s_branch", "s_cbranch")):
                offset = int(ops[0].split()[0])
                there = at[address + 4 + 4 * (offset - 65536 if offset >= 32768 else offset)]
                after = [there] if name == "s_branch" else after + [there]
            elif name in ("s_endpgm", "s_setpc_b64"):
                after = []
            self.next.append(after)

    def states(self, i):
        name, ops = self.code[i][1], self.code[i][2]
        return int(ops[0], 0) + 1 if name == "s_nop" else 1

    def matrix(self, i):
        return self.code[i][1].startswith("v_mfma")

    def follow(self, start, limit, see):
        """calls see(index) for every instruction fewer than `limit` wait states behind `start`; see returns True to stop there"""
        best, work = {}, [(n, 0) for n in self.next[start]]
        while work:
            i, passed = work.pop()
            if passed >= limit or best.get(i, limit) <= passed:
                continue
            best[i] = passed
            if not see(i):
                work += [(n, passed + self.states(i)) for n in self.next[i]]


def violations(code):
    c, bad, products = Code(code), [], 0
    for i, (_, name, _) in enumerate(code):
        if c.matrix(i):
            products += 1
            sums = c.used[i][0]

            def see(j, sums=sums, i=i):
                if not c.touched[j] & sums:
                    return False
                if c.matrix(j) and c.used[j][0] == sums and c.used[j][3] == sums and not (c.used[j][1] | c.used[j][2]) & sums:
                    return True   # goes on with them
                bad.append((i, j))
                return True

            c.follow(i, BEHIND, see)
        elif name.startswith("v_") and c.used[i]:
            written = c.used[i][0]

            def see(j, written=written, i=i):
                if c.matrix(j) and c.touched[j] & written:
                    bad.append((i, j))
                return False

            c.follow(i, BEFORE, see)
    return products, bad


def test_distances_around_the_products_of_the_tile_kernels(tmp_path):
    from geo_amd import _native
    found = {name: code for name, code in kernels(_native.lib_path(), tmp_path).items() if "k_tilesI" in name and code}
    assert len(found) == 6   # three tiles, two types
    for name, code in found.items():
        products, bad = violations(code)
        assert products >= 8, name
        assert not bad, (name, [(code[i], code[j]) for i, j in bad[:3]])


def test_the_check_sees_what_it_is_for():
    def at(*lines):
        return [(4 * i, l.split()[0], [o.strip() for o in l[len(l.split()[0]):].split(",")]) for i, l in enumerate(lines)]

    product = "v_mfma_i32_16x16x64_i8 a[0:3], v[0:3], v[4:7], a[0:3]"
    assert violations(at(product, product, "s_nop 15", "s_nop 3", "v_accvgpr_read_b32 v9, a2", "s_endpgm ")) == (2, [])
    assert violations(at(product, "s_nop 15", "v_accvgpr_read_b32 v9, a2", "s_endpgm "))[1] == [(0, 2)]
    assert violations(at("v_mov_b32_e32 v5, v9", "s_nop 0", product, "s_endpgm "))[1] == [(0, 2)]
    assert violations(at("v_mov_b32_e32 v5, v9", "s_nop 1", product, "s_endpgm "))[1] == []
    # over a branch back: the read stands in front of the product in the text
    assert violations(at("v_accvgpr_read_b32 v9, a1", "s_nop 1", product, "s_cbranch_scc1 65532", "s_endpgm "))[1] == [(2, 0)]
