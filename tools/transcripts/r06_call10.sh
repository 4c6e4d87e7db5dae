#!/bin/bash
# round 6, call 10: corrected GEMM workgroup timeline (its first part, the DDP overlap model with a communication stream of high priority, is taken out:
# streams of different priorities side by side have hung on this part)
cd "$GRAFT_REPO_ROOT"; export TMPDIR=/tmp
O=gpurun_out
tools/_bin/gemm_probe > $O/r06j_gemm_timeline.txt 2>&1
grep -v "k-block lengths" $O/r06j_gemm_timeline.txt | cut -c1-400
