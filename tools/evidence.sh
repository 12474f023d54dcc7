#!/bin/bash
# The evidence DESIGN.md's measurement table is made from: one machine, ONE library build (the counter summaries are stamped with its source id;
# bench.py quotes them only for that build): bench lines + rocprofv3 kernel traces for the main configurations with the mean over the TIMED
# dispatches taken from the trace (tools/trace_timed_mean.py), counter passes for them, the other shapes' lines, the host paths.
# Run from the repository's root on a machine with the GPU; writes gpurun_out/evidence, which tools/install_evidence.py puts in place.
# Every step has a time limit, and the first that fails ends the run.
set -eu
R=$PWD
O=$R/gpurun_out/evidence
mkdir -p "$O"
export TMPDIR=/tmp
bench() { local out=$1; shift; echo "bench $*"; timeout -k 10 150 python3 "$R/bench.py" "$@" > "$O/$out" 2> "$O/$out.err" || { tail -5 "$O/$out.err"; exit 1; }; }
for w in cfg2 cfg3 cfg4; do
  echo "trace $w"
  (cd /tmp && timeout -s KILL 150 rocprofv3 --kernel-trace --stats --output-format csv -d "$O/trace_$w" -- python3 "$R/bench.py" --workload $w --no-cpu-baseline --no-host-paths --no-n1-reference > "$O/trace_$w.json" 2> "$O/trace_$w.err")
  f=$(find "$O/trace_$w" -name "*kernel_stats.csv" | sed -n 1p); cp "$f" "$O/kernel_stats_$w.csv"
  t=$(find "$O/trace_$w" -name "*kernel_trace.csv" | sed -n 1p); sed -n 1,6p "$t" > "$O/kernel_trace_head_$w.csv"
  python3 "$R/tools/trace_timed_mean.py" "$t" "$O/trace_$w.json" >> "$O/trace_timed_means.log" 2>&1
  rm -rf "$O/trace_$w"
done
for w in cfg2 cfg3 cfg4 hq48 hq44 dn8; do
  echo "counters $w"
  bash "$R/tools/pmc_passes.sh" "$O/pmc_$w" --workload $w > "$O/pmc_$w.log" 2>&1 || { tail -5 "$O/pmc_$w.log"; exit 1; }
  cp "$O/pmc_$w/pmc_summary.txt" "$R/profiles/evidence_${w}_pmc_summary.txt"
  cp "$O/pmc_$w/pmc_summary.txt" "$O/pmc_summary_$w.txt"
  rm -rf "$O/pmc_$w"
done
bench bench_cfg2.json
bench bench_cfg2_steps20.json --steps 20 --warmup 3
bench bench_cfg3.json --workload cfg3
bench bench_cfg4.json --workload cfg4
for w in cfg5 hq48 hq44 dn8 dn2 dn6x dn21 dn32 up12 ch16 mono dn1; do bench bench_$w.json --workload $w --no-cpu-baseline --no-host-paths; done
bench bench_cfg2_s16.json --workload cfg2 --s16 --no-cpu-baseline
echo "host paths"; timeout -k 10 150 python3 tools/host_path_rate.py > "$O/host_paths.log" 2>&1
rm -f "$O"/*.err
