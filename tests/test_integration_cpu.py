"""The Rust declarations of the integration guide against the C header."""
import os
import re

from conftest import ROOT


def _rust():
    text = open(os.path.join(ROOT, "INTEGRATION.md"), encoding="utf-8").read()
    return [b for b in re.findall(r"```rust\n(.*?)```", text, re.S) if 'extern "C"' in b][0]


def _header():
    text = open(os.path.join(ROOT, "include", "riallm_cuda.h"), encoding="utf-8").read()
    return re.sub(r"/\*.*?\*/", "", text, flags=re.S)


def test_link_attribute_names_the_library_of_the_extern_block():
    lines = [x.strip() for x in _rust().splitlines() if x.strip()]
    at = [i for i, x in enumerate(lines) if x.startswith("#[link(")]
    assert len(at) == 1 and lines[at[0] + 1] == 'extern "C" {'


def test_every_entry_point_is_declared():
    rust = set(re.findall(r"pub fn (riallm_\w+)\(", _rust()))
    c = set(re.findall(r"\b(riallm_\w+)\s*\(", _header()))
    assert rust and rust <= c and {x for x in c if x.startswith("riallm_cuda_")} <= rust


def test_argument_structures_have_the_headers_fields():
    names = {"riallm_rope_paged_append_args": "RopePagedAppendArgs", "riallm_paged_attention_args": "PagedAttentionArgs",
             "riallm_verify_draft_args": "VerifyDraftArgs"}
    kinds = {"int32_t": "i32", "int64_t": "i64", "float": "f32", "void": "c_void"}
    for c_name, rust_name in names.items():
        body = re.search(r"typedef struct %s \{(.*?)\}" % c_name, _header(), re.S).group(1)
        want = []
        for decl in filter(None, (x.strip() for x in body.split(";"))):
            const, kind, rest = re.match(r"(const )?(\w+)(.*)", decl).groups()
            for name in rest.split(","):
                star = "*" in name
                want.append((name.strip("* ").lower(), ("*const " if const else "*mut ") * star + kinds[kind]))
        body = re.search(r"#\[repr\(C\)\]\npub struct %s \{(.*?)\n\}" % rust_name, _rust(), re.S).group(1)
        assert re.findall(r"pub (\w+): ([^,]+),", body) == want, rust_name
