#!/usr/bin/env python3
"""The operators over channels (yolo_amd.ops.layer_norm ... linear_i8) under rocprofv3:

    row_profile.py count                -> number of cases: those of perf/operators.py and a few more
    row_profile.py run <i>              -> case i, 24 calls over three sets of inputs (the program that the profiler runs)
    row_profile.py trace <dir>          -> per case and kernel the duration, from <dir>/t<i>/t_kernel_trace.csv (CSV on stdout)
    row_profile.py counters <dir>       -> per case and kernel the means of the counters, from <dir>/c<i><pass>/*.csv (JSON)

tools/profile_rows.sh takes both.  The summaries carry the hash of the kernel sources, as those of tools/rocprof_summary.py do.
"""
import collections
import csv
import glob
import importlib.util
import json
import os
import re
import statistics
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
CALLS = 24


def cases():
    spec = importlib.util.spec_from_file_location("operators", os.path.join(ROOT, "perf", "operators.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    m.own = True
    more = [dict(op="quant", rows=23104, c=2048, x="bf16", name="quantisation 23104 x 2048"),
            dict(op="ln_quant", rows=23104, c=2048, x="bf16", name="norm + quantisation 23104 x 2048"),
            dict(op="memory", rows=102400, k=256, n=1024, name="product, rows from memory")]
    return m, m.listed() + more


def describe(c):
    sizes = f"{c['rows']} x {c['c']}" if "c" in c else f"{c['rows']} x {c['k']} -> {c['n']}"
    return f"{c['name']} ({sizes}{' ' + c['x'] if 'x' in c else ''})"


def run(i):
    import torch
    from yolo_amd import ops
    m, all_cases = cases()
    c = all_cases[i]
    if c["op"] in ("quant", "ln_quant"):
        states = [torch.randn(c["rows"], c["c"], device="cuda").bfloat16() for _ in range(3)]
        w, b = torch.randn(2, c["c"], device="cuda")
        call = ops.quantize_rows if c["op"] == "quant" else lambda x: ops.layer_norm_quantize(x, w, b)
    elif c["op"] == "memory":
        byte = lambda *s: torch.randint(-128, 128, s, device="cuda", dtype=torch.int8)
        lin = ops.LinearI8(byte(c["n"], c["k"]), torch.rand(c["n"], device="cuda") * 0.01, torch.randn(c["n"], device="cuda"))
        s = torch.rand(c["rows"], device="cuda") * 0.01
        states = [byte(c["rows"], c["k"]) for _ in range(3)]
        call = lambda q: ops.matmul_i8(q, s, lin, act="silu")
    else:
        states, call = [m.prepare(c, k) for k in range(3)], m.run
    torch.cuda.synchronize()
    for k in range(CALLS):
        call(states[k % 3])
    torch.cuda.synchronize()
    print("done", describe(c), flush=True)


def kernel(name):
    """Short name of one of the operators' kernels with its template arguments, or None."""
    m = re.search(r"(row_norm_kernel|norm_grad_kernel|norm_grad_sum_kernel|tile_kernel|few_rows_kernel|few_float_rows_kernel|align_rows_kernel)", name)
    if not m or "ydet" not in name:
        return None
    k, rest = m.group(1), name[m.end():]
    if name.startswith("_Z"):
        args = [v if v else ("bf16" if t == "DF16b" else "fp32") for t, v in re.findall(r"(DF16b|f|L[ib](\d+)E)", rest[1:rest.find("EEv") + 1])]
    else:
        args = [a.strip().replace("__bf16", "bf16").replace("bool _Accum", "bf16").replace("float", "fp32") for a in rest[1:rest.find(">(")].split(",")]
    if args[1:3] == ["int", "E"]:       # (the demangler's reading of a number behind bf16: the two sides of the outputs are equal)
        args[1:3] = args[3:4]
    if k == "row_norm_kernel":
        return f"{k}<{('', 'norm', 'quantise', 'norm + quantise')[int(args[0])]}; {args[1]}; {args[3]} lanes x {args[4]} pieces; {args[5]} rows>"
    if k == "norm_grad_kernel":
        return f"{k}<{args[0]}; {args[2]} lanes x {args[3]} pieces; {args[4]} rows>"
    if k == "tile_kernel":
        return f"{k}<{args[0]} out; {args[1]} channels x {args[2]} pixels; {args[5]} stages>"
    if k == "few_rows_kernel":
        return f"{k}<{args[0]} out; {16 * int(args[1])} x {16 * int(args[2])}; {args[3]} waves>"
    if k == "few_float_rows_kernel":
        return f"{k}<{args[0]} out; {args[1]} rows>"
    return k


def csrc_hash():
    from bench import csrc_hash as h
    return h()


def trace(d):
    print(f"# rocprofv3 --kernel-trace -- python3 tools/row_profile.py run <case> (tools/profile_rows.sh); {CALLS} calls over three sets of inputs; "
          f"csrc_sha1 {csrc_hash()}")
    print("case,kernel,workgroups,calls,median_us,min_us")
    for i, c in enumerate(cases()[1]):
        per = collections.OrderedDict()
        with open(os.path.join(d, f"t{i}", "t_kernel_trace.csv")) as fh:
            for r in sorted(csv.DictReader(fh), key=lambda r: int(r["Start_Timestamp"])):
                k = kernel(r["Kernel_Name"])
                if k:
                    key = k, int(r["Grid_Size_X"]) // int(r["Workgroup_Size_X"])
                    per.setdefault(key, []).append((int(r["End_Timestamp"]) - int(r["Start_Timestamp"])) / 1e3)
        for (k, groups), v in per.items():
            if len(v) >= CALLS:       # (not the quantisation of a layer's weights)
                print(f'"{describe(c)}","{k}",{groups},{len(v)},{statistics.median(v):.2f},{min(v):.2f}')


def counters(d):
    out = collections.OrderedDict()
    for i, c in enumerate(cases()[1]):
        per = {}
        for path in sorted(glob.glob(os.path.join(d, f"c{i}[a-z]", "*counter_collection.csv"))):
            with open(path) as fh:
                for r in csv.DictReader(fh):
                    k = kernel(r["Kernel_Name"])
                    if k:
                        per.setdefault(k, {}).setdefault(r["Counter_Name"], []).append(float(r["Counter_Value"]))
        for k, cs in per.items():
            if max(map(len, cs.values())) < CALLS:
                continue
            v = {n: round(statistics.median(x), 1) for n, x in cs.items()}
            if v.get("GRBM_GUI_ACTIVE"):
                simd = v["GRBM_GUI_ACTIVE"] / 8.0 * 1024.0        # SIMD-cycles of the launch; SQ_ACTIVE_* tick once in four cycles
                for n, key, per_tick in (("SQ_ACTIVE_INST_VALU", "valu_active_frac", 4), ("SQ_VALU_MFMA_BUSY_CYCLES", "mfma_busy_frac", 1),
                                         ("SQ_ACTIVE_INST_VMEM", "vmem_inst_active_frac", 4), ("SQ_WAVE_CYCLES", "waves_per_simd", 4)):
                    if n in v:
                        v[key] = round(v[n] * per_tick / simd, 4)
            if "FETCH_SIZE" in v:
                v["read_mb"] = round(2 * v["FETCH_SIZE"] / 1e3 * 1.024, 1)       # (kilobytes; 128-byte requests are tallied at 64)
            if "WRITE_SIZE" in v:
                v["written_mb"] = round(v["WRITE_SIZE"] / 1e3 * 1.024, 1)
            out.setdefault(describe(c), {})[k] = v
    print(json.dumps(dict(source="rocprofv3 --pmc passes of `python3 tools/row_profile.py run <case>` (tools/profile_rows.sh); medians over launches; "
                                 "GRBM_GUI_ACTIVE is the sum over the 8 XCDs", csrc_sha1=csrc_hash(), cases=out), indent=1))


if __name__ == "__main__":
    what = sys.argv[1]
    if what == "count":
        print(len(cases()[1]))
    elif what == "run":
        run(int(sys.argv[2]))
    else:
        (trace if what == "trace" else counters)(sys.argv[2])
