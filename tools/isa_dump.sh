#!/bin/bash
# Cross-compile one csrc/*.hip file to gfx950 assembly (no GPU needed) and print resource usage; the .s lands in /tmp.
f=${1:-gemm_w4.hip}
cd /root/repo/open_flamingo_amd/csrc
flags=$(PYTHONPATH=/root/repo python -c "from open_flamingo_amd.csrc import build as b; print(' '.join(b.FLAGS))")
/opt/rocm/bin/hipcc $flags -S --cuda-device-only $f -o /tmp/${f%.hip}.s -Rpass-analysis=kernel-resource-usage 2>&1 | grep -E "VGPRs:|AGPRs:|Scratch|error|Occupancy" | sort | uniq -c
