#!/bin/bash
# Round 5, experiment c: as b, without the harness's own tail (special rows), timeline symbol set before the first launch.
ROOT=${GRAFT_REPO_ROOT:-/root/repo}
O=$ROOT/gpurun_out/r05c
mkdir -p $O
cd $ROOT
{
timeout 120 tools/ubench/bin/qb_B4 16 50 B4 4
QB_SPECIAL=1 timeout 120 tools/ubench/bin/qb_B4 16 10 B4special 4
timeout 120 tools/ubench/bin/qb_B4tl 16 20 B4tl 4
} 2>&1 | tee $O/log.txt
