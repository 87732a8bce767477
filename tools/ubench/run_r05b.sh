#!/bin/bash
# Round 5, experiment b: warmed-up timings of fft_quad_kernel (B4) and its phase timeline.
ROOT=${GRAFT_REPO_ROOT:-/root/repo}
O=$ROOT/gpurun_out/r05b
mkdir -p $O
cd $ROOT
{
timeout 120 tools/ubench/bin/qb_B4 16 50 B4 4
timeout 120 tools/ubench/bin/qb_B4tl 16 20 B4tl 4
} 2>&1 | tee $O/log.txt
