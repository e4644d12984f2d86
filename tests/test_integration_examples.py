"""The C examples of the integration notes compile against the header as a caller would compile them
(-Wall -Wextra -Werror), structs are initialised by member name where members of one type stand side by
side, and the Zig declarations there have the header's parameters and members, one by one."""
import os
import re
import subprocess

import pytest

from tests.conftest import ROOT

with open(os.path.join(ROOT, "INTEGRATION.md")) as f:
    NOTES = f.read()
with open(os.path.join(ROOT, "include", "zwgpu.h")) as f:
    HEADER = re.sub(r"/\*.*?\*/", "", f.read(), flags=re.S)

# what the text around an example says is there already
THERE = """
#include <stddef.h>
#include <stdint.h>
#include <string.h>
#include "zwgpu.h"
static int cudaMalloc(void** p, size_t n) { (void)p; (void)n; return 0; }
static int cudaMemcpyAsync(void* d, const void* s, size_t n, int k, void* st) { (void)d; (void)s; (void)n; (void)k; (void)st; return 0; }
static int cudaMemcpy2DAsync(void* d, size_t dp, const void* s, size_t sp, size_t w, size_t h, int k, void* st)
{ (void)d; (void)dp; (void)s; (void)sp; (void)w; (void)h; (void)k; (void)st; return 0; }
enum { cudaMemcpyHostToDevice = 1, cudaMemcpyDeviceToDevice = 3 };
"""
LLM = "zwg_llm_state* llm, size_t n_past, size_t n, size_t n_seq, void* stream, float* x, float* logits, int32_t* prompt_chunk, " \
      "int32_t* recent, int32_t* next"
EXAMPLES = [  # the text it starts with, what is there
    ("zwg_init(0);\nzwg_llm_state* llm;", "size_t n_layer, size_t n_seq, size_t n_windows, size_t n_past, size_t n, size_t layer, "
     "size_t window, float* q, float* k, float* v, float* attn_out, float* cross_k, float* cross_v, float* k_new, float* v_new, "
     "float* out, float* q_cross, float* out_cross, void* stream"),
    ("size_t n_len = zwg_mel_frames", "size_t n_samples, size_t n_windows, const float* d_samples, const float* d_filters, float* d_mel, "
     "void* d_mel_scratch, const uint16_t* d_conv1_taps, const float* d_conv1_b, const uint16_t* d_conv2_taps, const float* d_conv2_b, "
     "const float* d_pos, const zwg_enc_layer_weights* host_layer_array, const float* d_lnw, const float* d_lnb, float* d_enc, void* d_scratch, "
     "void* stream"),
    ("zwg_llm_layer_weights lw[28];", LLM + ", zwg_q8_mat embd, const float* output_norm, void* scratch, int max_new"),
    ("zwg_llm_state_create_kv8(", LLM + ", zwg_llm_weights w, void* scratch, size_t bytes, const float* cos, const float* sin, "
     "size_t max_new, size_t s, const int32_t* bias_ids, const float* bias, size_t n_bias, const uint32_t* allow"),
    ("zwg_seqs s = {", "size_t n_seq, size_t n, size_t n_past, const int32_t* past, const int32_t* count, const int32_t* first, "
     "zwg_rope_tables tables, zwg_rows q, zwg_rows k, zwg_rows v, zwg_rows out, zwg_kv8 cache, void* ws, size_t ws_bytes, void* stream"),
    ("zwg_whisper_rules rules;", "zwg_dec_state* dec, zwg_dec_weights weights, size_t n_windows, size_t b, size_t n_prompt, size_t cap, "
     "const int32_t* seek, const int32_t* n_len_org, zwg_whisper_window* win_h, zwg_whisper_window* win, float** enc_out, "
     "const int32_t* prompt, int32_t* tokens, int32_t* tids, void* scratch, void* stream"),
]


def blocks(language):
    return re.findall(r"```" + language + r"\n(.*?)```", NOTES, flags=re.S)


def test_every_example_is_here():
    assert len(blocks("c")) == len(EXAMPLES)


@pytest.mark.parametrize("starts,there", EXAMPLES, ids=[re.sub(r"\W+", "_", e[0])[:24] for e in EXAMPLES])
def test_c_example(tmp_path, starts, there):
    code, = [b for b in blocks("c") if b.startswith(starts)]
    src = tmp_path / "example.c"
    src.write_text(f"{THERE}\nvoid example({there});\nvoid example({there})\n{{\n{code}\n}}\n")
    out = subprocess.run(["gcc", "-std=c11", "-Wall", "-Wextra", "-Werror", "-Wno-missing-field-initializers", "-Wno-unused-function", "-Wno-unused-parameter",
                          "-Wno-unused-variable", "-Wno-unused-but-set-variable", "-fsyntax-only", "-I", os.path.join(ROOT, "include"),
                          str(src)], capture_output=True, text=True)
    assert out.returncode == 0, out.stderr


def test_logit_rules_are_initialised_by_name():
    """recent_stride, n_recent and the like are all size_t: a compiler takes them in any order."""
    for code in (re.sub(r"/\*.*?\*/", "", b, flags=re.S) for b in blocks("c")):
        for init in re.findall(r"zwg_logit_rules \w+ = \{(.*?)\}", code, flags=re.S):
            assert all(part.strip().startswith(".") for part in init.split(",") if part.strip()), init


KINDS = {"usize": "size_t", "c_int": "int", "f32": "float", "f64": "double", "i32": "int32_t", "u32": "uint32_t", "i8": "int8_t",
         "u16": "uint16_t", "u8": "char"}


def header_params(name):
    args = re.search(r"ZWG_API [\w\s*]+?\b" + name + r"\(([^)]*)\)", HEADER).group(1)
    return [] if args.strip() in ("", "void") else [a.strip() for a in args.split(",")]


def same_kind(zig, c):
    """A Zig type against a C parameter or member: scalars by name, pointers as pointers, a struct's by itself."""
    pointer = zig.startswith(("*", "?*", "[*", "?[*"))
    if pointer != ("*" in c):
        return False
    base = re.sub(r"^\??(\*|\[\*\])(const )?", "", zig)
    if pointer and base in ("anyopaque",):
        return True
    return base not in KINDS or re.search(r"\b" + KINDS[base] + r"\b", c) is not None


def test_zig_functions():
    seen = 0
    for code in blocks("zig"):
        for name, args in re.findall(r'extern "c" fn (zwg_\w+)\(([^)]*)\)', code):
            zig = [a.split(":", 1)[1].strip() for a in args.split(",") if a.strip()]
            want = header_params(name)
            assert len(zig) == len(want), (name, zig, want)
            for z, c in zip(zig, want):
                assert same_kind(z, c), (name, z, c)
            seen += 1
    assert seen >= 9


def header_members(name):
    body = re.search(r"typedef struct " + name + r" \{(.*?)\}", HEADER, flags=re.S).group(1)
    out = []
    for line in body.split(";"):
        if line.strip():
            kind, names = re.match(r"\s*((?:const )?\w+\s*\**)\s*(.*)", line.strip(), flags=re.S).groups()
            out += [(re.sub(r"\W", "", n), kind) for n in names.split(",")]
    return out


@pytest.mark.parametrize("zig,c", [("EncWeights", "zwg_enc_weights"), ("EncLayer", "zwg_enc_layer_weights"), ("Seqs", "zwg_seqs"),
                                   ("Rows", "zwg_rows"), ("RopeTables", "zwg_rope_tables"), ("Kv8", "zwg_kv8"),
                                   ("LogitRules", "zwg_logit_rules"), ("WhisperWindow", "zwg_whisper_window")])
def test_zig_structs(zig, c):
    body, = re.findall(r"const " + zig + r" = extern struct \{(.*?)\}", "\n".join(blocks("zig")), flags=re.S)
    got = [tuple(x.strip() for x in m.split(":", 1)) for m in re.sub(r"//.*", "", body).split(",") if m.strip()]
    want = header_members(c)
    assert [n for n, _ in got] == [n for n, _ in want]
    for (n, z), (_, k) in zip(got, want):
        assert same_kind(z, k), (n, z, k)


def test_the_8_bit_step_is_declared_for_zig():
    declared = set(re.findall(r'extern "c" fn (zwg_\w+)\(', "\n".join(blocks("zig"))))
    assert {"zwg_rope", "zwg_kv8_append", "zwg_kv8_read", "zwg_kv8_attn_workspace", "zwg_kv8_attn", "zwg_llm_logits",
            "zwg_llm_state_create_kv8", "zwg_llm_state_kv8", "zwg_llm_state_set_rope"} <= declared
