#!/usr/bin/env python
"""Generates diffbir_amd/csrc/plan_dispatch.inc — the switch dbir_plan_run uses to call a recorded operator entry point with
its recorded arguments — from the one signature table the ctypes binding uses (diffbir_amd/native.py SIGNATURES), so the
recorder (diffbir_amd/plan.py) and the replayer cannot disagree about argument order or types.  Every recordable entry point
takes `void* stream` last; ints / long longs / floats / pointers travel in 8-byte dbir_arg slots.  The calls go through
function pointers with generic parameter types (int, long long, float, void*): ABI-identical to the declared prototypes.
tests/test_plan_cpu.py checks that the committed .inc equals this script's output."""
import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
from diffbir_amd import native  # noqa: E402

OUT = os.path.join(ROOT, "diffbir_amd", "csrc", "plan_dispatch.inc")
NOT_RECORDABLE = {"dbir_groupnorm_nchunk", "dbir_xf_tile_bytes", "dbir_xf_head_tiles", "dbir_xf_tail_tiles", "dbir_xf_geometry", "dbir_xf2_geometry",
                  "dbir_abi_version", "dbir_set_option", "dbir_cldm_forward",
                  # training operators: not part of a network evaluation (ops.py refuses them while one is recorded)
                  "dbir_attention_fwd", "dbir_attention_bwd", "dbir_layernorm_fwd", "dbir_layernorm_bwd", "dbir_embedding_fwd", "dbir_embedding_bwd"}
CT = {native._I: ("int", "(int)a[{k}].i"), native._LL: ("long long", "a[{k}].i"), native._F: ("float", "(float)a[{k}].f"),
      native._P: ("void*", "a[{k}].p")}


def recordable():
    return sorted(n for n, sig in native.SIGNATURES.items()
                  if n not in NOT_RECORDABLE and not n.startswith("dbir_plan_") and sig and sig[-1] is native._P)


def generate() -> str:
    names = recordable()
    out = ["// GENERATED by tools/gen_plan_dispatch.py from diffbir_amd/native.py SIGNATURES — do not edit.",
           f"static const int kPlanFnCount = {len(names)};",
           "static const char* const kPlanFnNames[] = {" + ", ".join(f'"{n}"' for n in names) + "};",
           "static const int kPlanFnArgs[] = {" + ", ".join(str(len(native.SIGNATURES[n]) - 1) for n in names) + "};",
           "static int plan_dispatch(int fn, const dbir_arg* a, const char* blob, void* stream) {", "  switch (fn) {"]
    for i, n in enumerate(names):
        sig = native.SIGNATURES[n]
        if n == "dbir_gemm":
            out += [f"    case {i}: {{  // {n}: the descriptor travels by value in the plan's blob",
                    "      dbir_gemm_desc d;", "      memcpy(&d, blob + a[0].i, sizeof(d));",
                    "      return dbir_gemm(&d, stream);", "    }"]
            continue
        types = ", ".join(CT[t][0] for t in sig[:-1]) + ", void*"
        args = ", ".join(CT[t][1].format(k=k) for k, t in enumerate(sig[:-1])) + ", stream"
        out += [f"    case {i}: {{  // {n}", f"      typedef int (*fn_t)({types});",
                f"      return reinterpret_cast<fn_t>(reinterpret_cast<void*>(&{n}))({args});", "    }"]
    out += ["  }", '  dbir_set_error("dbir_plan_run: bad function index %d", fn);', "  return DBIR_ERR_ARG;", "}", ""]
    return "\n".join(out)


if __name__ == "__main__":
    with open(OUT, "w") as f:
        f.write(generate())
    print(OUT, len(recordable()), "entry points")
