"""The tree attention's O lives in accumulation registers that inline-asm MFMAs write: the
compiler does not know their latency, so whatever it does itself with such a register has to
come behind the waits of `acc_settle`. (With twelve waves some other registers do spill, outside
the loop over tiles or where a sum's reference moves.)"""
import re
import subprocess

import __graft_entry__ as ge


def agprs(operand):
    """The accumulation registers that one operand names."""
    m = re.fullmatch(r"a\[(\d+):(\d+)\]|a(\d+)", operand)
    if not m:
        return set()
    return {int(m[3])} if m[3] else set(range(int(m[1]), int(m[2]) + 1))


def lines_of(body):
    """(the inner loop that it is in, in an asm block, mnemonic, operands) of each instruction."""
    app, label, loop = False, "", ""
    for line in body.split("\n"):
        line = line.strip()
        if line.startswith(";;#ASMSTART"):
            app = True
        elif line.startswith(";;#ASMEND"):
            app = False
        if m := re.match(r"\.L(BB\w+):", line):
            label, loop = m[1], ""
        elif line.startswith("; %bb"):
            loop = ""
        if m := re.search(r"in Loop: Header=(BB\w+) Depth=[2-9]", line):
            loop = m[1]
        elif re.search(r"Loop Header: Depth=[2-9]", line):
            loop = label
        line = line.split(";")[0].strip()
        if line and not line.startswith(".") and not line.endswith(":"):
            op, _, rest = line.partition(" ")
            yield loop, app, op, [x.strip() for x in rest.split(",")]


def test_nothing_reads_an_accumulator_ahead_of_its_waits(tmp_path):
    builder = ge._load_builder()
    csrc = next(p for p in ge.PKG_DIR.rglob("attn_tree.hip"))
    out = tmp_path / "out.s"
    subprocess.run([builder.hipcc(), *builder.HIPCC_FLAGS, *builder.FILE_FLAGS["attn_tree"],
                    "--cuda-device-only", "-S", str(csrc), "-o", str(out)],
                   check=True, capture_output=True, timeout=300)
    text, found = out.read_text(), 0
    for name in re.findall(r"^(_ZN\S*tree_attn_kernel\S*):", text, flags=re.M):
        body = text[text.index(f"\n{name}:"):]
        rows = list(lines_of(body[:body.index(".Lfunc_end")]))
        products = [(loop, ops) for loop, app, op, ops in rows if app and op.startswith("v_mfma")]
        O = set().union(*(agprs(ops[0]) for _, ops in products))
        tiles = {loop for loop, _ in products} - {""}
        assert len(O) == 64 and tiles, f"{name}: {len(O)} accumulators"
        nops, settled, last = 0, True, ""
        for loop, app, op, ops in rows:
            if (loop in tiles and loop != last) or (app and op.startswith("v_mfma")):
                settled = False
            last = loop
            nops = nops + 1 if app and op == "s_nop" and ops == ["7"] else 0
            settled = settled or nops == 3
            reads = ops if op.startswith(("global_store", "scratch_store", "ds_write", "buffer_store")) else ops[1:]
            if not app and not settled and any(agprs(x) & O for x in reads):
                raise AssertionError(f"{name}: {op} {', '.join(ops)} reads an accumulator that may be in flight")
        found += 1
    assert found >= 5
