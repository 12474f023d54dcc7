#!/usr/bin/env python3
"""Copies gpurun_out/evidence/* (tools/evidence.sh) into profiles/ under evidence_ names and rewrites the measurement table of DESIGN.md
section 5 (between the MEASUREMENTS markers) from them."""
import json, os, re, shutil
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
O, P = os.path.join(ROOT, "gpurun_out", "evidence"), os.path.join(ROOT, "profiles")
FULL = ("cfg2", "cfg2_steps20", "cfg5", "cfg4", "cfg3", "hq48", "hq44", "dn8", "cfg2_s16")
MORE = ("dn2", "mono", "dn1", "dn6x", "dn21", "dn32", "up12", "ch16")

for f in sorted(os.listdir(O)):
    if f.endswith((".json", ".csv", ".log", ".txt")) and not f.startswith(("trace_cfg", "pmc_cfg", "pmc_hq", "pmc_dn")):
        dst = re.sub(r"^pmc_summary_(\w+)\.txt$", r"\1_pmc_summary.txt", f)
        text = "".join(l for l in open(os.path.join(O, f)) if "amdgpu.ids" not in l)
        open(os.path.join(P, "evidence_" + dst), "w").write(text)


def line(w):
    return json.loads([x for x in open(os.path.join(P, "evidence_bench_%s.json" % w)) if x.startswith("{")][0])


timed = {}
for l in open(os.path.join(P, "evidence_trace_timed_means.log")):
    m = re.match(r"(\w+)[^:]*: (\d+) dispatches.*all: mean ([\d.]+) us; timed region \[\d+, \d+\): mean ([\d.]+) us", l)
    if m:
        timed[m.group(1)] = (int(m.group(2)), float(m.group(3)), float(m.group(4)))
k = lambda x: "{:,.0f}".format(round(x, -2))
rows = ["| workload | kernel | output Msamples/s | µs per launch (`bench.py`, K timed launches behind the lead-in; rocprofv3 kernel trace of the same command) | GB/s (algorithmic) | frac of 8 TB/s | VALU issuing | HBM traffic ÷ algorithmic |",
        "|---|---|---:|---:|---:|---:|---:|---:|"]
names = {"cfg2": "cfg 2 stereo 44.1→48 kHz, 3 lobes, 10 min (default, the headline)", "cfg2_steps20": "the same with `--steps 20 --warmup 3`", "cfg5": "cfg 5 same, 1 hour as one launch",
         "cfg4": "cfg 4 8-ch 48→44.1 kHz, 10 min", "cfg3": "cfg 3 stereo 8→96 kHz, 8 lobes, 10 min", "hq48": "stereo 44.1→48 kHz, 8 lobes (`hq48`)", "hq44": "stereo 48→44.1 kHz, 8 lobes (`hq44`)",
         "dn8": "stereo 44.1→8 kHz, 33 slots (`dn8`)", "cfg2_s16": "cfg 2 with the opt-in int16 output (`--s16`)", "dn2": "stereo 48→44.1 kHz (`dn2`)", "mono": "mono 44.1→48 kHz (`mono`)", "dn1": "mono 48→44.1 kHz (`dn1`)",
         "dn6x": "stereo 48→8 kHz (`dn6x`)", "dn21": "stereo 2:1 (`dn21`)", "dn32": "stereo 3:2 (`dn32`)", "up12": "12 channels 44.1→48 kHz (`up12`)", "ch16": "16 channels 44.1→48 kHz (`ch16`)"}
for w in FULL + MORE:
    l = line(w)
    assert l.get("parity_full_stream") in (True, None), w
    r, v = l["roofline"], l.get("roofline_valu") or {}
    us = "%.1f" % (l["ms_per_step"] * 1e3)
    if w in timed:
        us += " (rocprofv3, the timed dispatches: %.1f; all %s: %.1f)" % (timed[w][2], "{:,}".format(timed[w][0]), timed[w][1])
    tr = (r["traffic"] / r["algorithmic_bytes_per_launch"]) if r.get("traffic") else None
    rows.append("| %s | `%s` | %s | %s | %s | **%.3f** | %s | %s |" % (names[w], r["kernel"], k(l["value"]), us, "{:,.0f}".format(r["achieved"]), r["frac"],
                "" if not v else "%.2f" % v["frac"], "" if tr is None else "%.3f" % tr))
c2 = line("cfg2")
cb = c2["cpu_baseline"]
rows.append("| reference C path on this box's host (`cpu_baseline`, kind \"%s\") | | %.0f on 1 core; %.0f on %d cores (oracle driver) | | | | | |" % (cb["kind"], cb["value"], cb["all_cores"]["value"], cb["all_cores"]["cores"]))
e2e, cbk, s1 = c2["end_to_end"], c2["callback_api"], c2["strong_curve_n1"]
stamp = open(os.path.join(P, "evidence_cfg2_pmc_summary.txt")).readline().split()[-1]
notes = ("\n(One box, one build - source id `%s`, which stamps the counter summaries `profiles/evidence_{cfg2,cfg3,cfg4,hq48,hq44,dn8}_pmc_summary.txt`; bench lines `profiles/evidence_bench_*.json`, rocprofv3 kernel "
         "stats `profiles/evidence_kernel_stats_*.csv`, `profiles/evidence_kernel_trace_head_*.csv`. `parity_full_stream` true in every int32 line. cfg 2 `end_to_end` pageable %.2f ms / page-locked %.2f ms, the "
         "reference's callback signature %.0f Msamples/s; `strong_curve_n1` (cfg 5 in the default line) %.1f us, %.3f.)" % (stamp, e2e["pageable_ms"], e2e["pinned_ms"], cbk["Msamples/s"], s1["ms_per_step"] * 1e3, s1["frac"]))
p = os.path.join(ROOT, "DESIGN.md")
s = open(p).read()
s = re.sub(r"<!-- MEASUREMENTS BEGIN.*?<!-- MEASUREMENTS END -->", lambda m: "<!-- MEASUREMENTS BEGIN (tools/install_evidence.py) -->\n" + "\n".join(rows) + "\n" + notes + "\n<!-- MEASUREMENTS END -->", s, flags=re.S)
open(p, "w").write(s)
print("\n".join(rows) + "\n" + notes)
