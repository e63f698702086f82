"""The OCaml stubs of the operators on a paged cache (ocaml/sarek-hip/Hip_attention.ml), read as text: symbols, signatures and the two
structures against include/sarek_hip.h."""
import os
import re

import pytest

import test_ocaml_veneer as veneer

STRUCTS = {"rotary_plan": "sarek_hip_rotary_plan", "kv_cache": "sarek_hip_kv_cache"}
TEXT = re.sub(r"\(\*.*?\*\)", "", open(os.path.join(veneer.OCAML, "Hip_attention.ml")).read(), flags=re.S)


@pytest.fixture(autouse=True)
def structs(monkeypatch):
    for var, name in STRUCTS.items():
        monkeypatch.setitem(veneer.OCAML_SCALARS, var, name)


def test_stubs_bind_the_header_with_its_signatures():
    protos, found = veneer.header_prototypes(), set()
    for m in re.finditer(r'bind\s+"(sarek_hip_\w+)"\s*\((.*?returning\s+\w+)\)', TEXT, flags=re.S):
        parts = [p.strip() for p in " ".join(m.group(2).split()).split("@->")]
        ret, args = protos[m.group(1)]
        assert veneer.squeeze(veneer.c_of_ocaml(parts[-1].replace("returning", ""))) == veneer.squeeze(ret), m.group(1)
        assert [veneer.squeeze(veneer.c_of_ocaml(a)) for a in parts[:-1]] == [veneer.squeeze(a) for a in args], m.group(1)
        found.add(m.group(1))
    assert found == {n for n in protos if re.match(r"sarek_hip_(rotary|kv_append|attention)", n)}


@pytest.mark.parametrize("var", STRUCTS)
def test_structures_follow_the_header(var):
    got = [(m.group(1), veneer.squeeze(veneer.c_of_ocaml(m.group(2)))) for m in re.finditer(r'field ' + var + r' "(\w+)" (\(ptr \w+\)|\w+)', TEXT)]
    want, body = [], re.search(r"typedef struct[^{]*\{([^}]*)\}\s*" + STRUCTS[var] + r"\s*;", veneer.header_text(), flags=re.S).group(1)
    for declaration in (" ".join(d.replace("const ", "").split()) for d in body.split(";") if d.strip()):
        base = declaration.split()[0]
        for name in declaration[len(base):].split(","):
            want.append((name.replace("*", "").strip(), base + "*" * name.count("*")))
    assert got == want and f"seal {var}" in TEXT
