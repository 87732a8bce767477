#!/bin/bash
# Evidence run on ONE box: the bench lines, rocprofv3 kernel stats and the separate PMC passes for both providers, the HBM-traffic
# file with its provenance, the default and driver-form lines quoting that traffic, the other BASELINE configs.  Every step that uses
# the GPU has its own time limit, and the first one that fails ends the run.
#   tools/profile_evidence.sh [lines|profile|configs ...]   (default: all three)
ROOT=${GRAFT_REPO_ROOT:-/root/repo}
O=$ROOT/gpurun_out/evidence
mkdir -p $O
export TMPDIR=/tmp
parts=${*:-lines profile configs}
bench() { out=$1; shift; cd $ROOT && timeout -k 10 240 python bench.py "$@" > $O/$out.json 2> $O/$out.err && echo "done $out"; }
prof() {  # prof <folder> <rocprofv3 options> -- <command>
  dir=$1; shift; mkdir -p $O/$dir; cd /tmp && timeout -s KILL 180 rocprofv3 "${@:1:$(($# - 1))}" --output-format csv -d $O/$dir -- ${!#} > $O/$dir.log 2>&1 && echo "done $dir"
}
SQ="SQ_WAVE_CYCLES SQ_BUSY_CYCLES SQ_INSTS_VALU SQ_ACTIVE_INST_VALU SQ_WAIT_INST_ANY SQ_WAIT_ANY SQ_ACTIVE_INST_ANY SQ_INSTS_LDS"
lines() {
  bench bench_default && bench bench_generic --provider generic --no-cpu-baseline --no-alt && bench bench_per_cycle --no-batch --no-cpu-baseline --no-alt
}
profile() {
  for v in fast generic; do
    B="python3 $ROOT/bench.py --provider $v --no-cpu-baseline --no-alt --no-parity --min-time 0.05"
    prof $v/trace --kernel-trace --stats "$B" && prof $v/pmc_fetch --kernel-trace --pmc FETCH_SIZE "$B" && prof $v/pmc_write --kernel-trace --pmc WRITE_SIZE "$B" \
      && prof $v/pmc_sq --kernel-trace --pmc $SQ "$B" || return 1
    python3 $ROOT/tools/pmc_summary.py $O/$v > $O/pmc_counters_$v.txt && python3 $ROOT/tools/kstats.py $O/$v/trace > $O/kernel_stats_$v.txt || return 1
  done
  # the launch form of --steps 20: ring period 20, one 20-cycle launch per unit and region
  B="python3 $ROOT/bench.py --slots 20 --no-cpu-baseline --no-alt --no-parity --no-configs --no-host-fed --min-time 0.05"
  prof fast20/trace --kernel-trace --stats "$B" && prof fast20/pmc_fetch --kernel-trace --pmc FETCH_SIZE "$B" && prof fast20/pmc_write --kernel-trace --pmc WRITE_SIZE "$B" || return 1
  python3 $ROOT/tools/kstats.py $O/fast20/trace > $O/kernel_stats_fast_period20.txt || return 1
  rm -f $O/pmc_traffic.json
  cd $ROOT && python3 tools/pmc_summary.py $O/fast20 --traffic-json $O/pmc_traffic.json --provider fast --cycles 20 > $O/pmc_traffic.log \
    && python3 tools/pmc_summary.py $O/generic --traffic-json $O/pmc_traffic.json --provider generic --cycles 32 >> $O/pmc_traffic.log \
    && python3 tools/pmc_summary.py $O/fast --traffic-json $O/pmc_traffic.json --provider fast --cycles 32 >> $O/pmc_traffic.log || return 1
  cp $O/pmc_traffic.json $ROOT/profiles/pmc_traffic.json  # so that the lines below quote this run's own counters
  bench bench_default_with_traffic --no-cpu-baseline --no-alt --no-parity && bench bench_driver_form --steps 20 --warmup 5
}
configs() {
  cd $ROOT && timeout -k 10 240 python tools/bench_configs.py > $O/bench_configs.jsonl 2> $O/bench_configs.err && echo "done configs" \
    && timeout -k 10 120 python tools/bench_multi_fm.py 400 > $O/multi_fm.json 2>> $O/bench_configs.err \
    && timeout -k 10 120 python tools/bench_fir.py > $O/config_C3_fast_ab.json 2>> $O/bench_configs.err \
    && timeout -k 10 120 python tools/bench_c5_streams.py generic > $O/config_C5_streams.json 2>> $O/bench_configs.err \
    && timeout -k 10 120 python tools/bench_c5_streams.py fast > $O/config_C5_streams_fast.json 2>> $O/bench_configs.err || return 1
  for c in C3 C4 C5; do
    prof cfg_$c --kernel-trace --stats "python3 $ROOT/tools/bench_configs.py $c" && python3 $ROOT/tools/kstats.py $O/cfg_$c > $O/kernel_stats_config_$c.txt || return 1
  done
  prof fir --kernel-trace --stats "python3 $ROOT/tools/bench_fir.py" && python3 $ROOT/tools/kstats.py $O/fir > $O/kernel_stats_config_C3_fast.txt \
    && prof mfm --kernel-trace --stats "python3 $ROOT/tools/bench_multi_fm.py 200" && python3 $ROOT/tools/kstats.py $O/mfm > $O/kernel_stats_multi_fm.txt
}
rc=0
for p in $parts; do $p || { rc=$?; echo "$p failed: $rc"; break; }; done
find $O -name "*.db" -delete; find $O -name "*kernel_trace.csv" -delete; find $O -name "*counter_collection.csv" -size +8M -delete
exit $rc
