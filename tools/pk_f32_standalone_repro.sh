#!/bin/bash
# GPU box: the standalone packed-fp32-beside-MFMA reproduction at the machine's own settings.  Its aggressors differ in power as well as in
# instructions: mismatches that follow the instruction and not the power speak for a structural hazard and against voltage droop.
#   bash tools/pk_f32_standalone_repro.sh > gpurun_out/pk_repro.txt
/opt/rocm/bin/hipcc --offload-arch=gfx950 -O2 tools/pk_f32_standalone_repro.hip -o /tmp/pkrepro || exit 1
smi() { /opt/rocm/bin/rocm-smi --showclocks --showpower --csv 2>/dev/null | grep "^card" | head -1 | cut -d, -f1-14; }
echo "# idle: $(smi)"
/opt/rocm/bin/rocm-smi --showmaxpower 2>/dev/null | grep -i "max" | head -2
echo "## default power cap"
/tmp/pkrepro ${1:-400} &
PID=$!; sleep 4; echo "# during: $(smi)"; wait $PID
echo "# after: $(smi)"
