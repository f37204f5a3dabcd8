#!/bin/bash
# Kernel times and counters of the operators over channels, from the repository root: tools/profile_rows.sh <dir>
# Leaves <dir>/{t<case>,c<case><pass>}; afterwards
#   python3 tools/row_profile.py trace <dir> > profiles/row_operators_kernel_times.csv
#   python3 tools/row_profile.py counters <dir> > profiles/row_operators_counters.json
# Counters never share a run with a trace, nor more than one block's worth a pass.
set -e
out=$1
mkdir -p $out
export TMPDIR=/tmp
n=$(python3 tools/row_profile.py count)
for ((i = 0; i < n; i++)); do
  timeout -k 10 90 rocprofv3 --kernel-trace --output-format csv -d $out/t$i -o t -- python3 tools/row_profile.py run $i > $out/t$i.log 2>&1
  tail -1 $out/t$i.log
done
for ((i = 0; i < n; i++)); do
  timeout -s KILL 90 rocprofv3 --pmc SQ_WAVES SQ_WAVE_CYCLES SQ_WAIT_ANY SQ_ACTIVE_INST_ANY SQ_ACTIVE_INST_VALU SQ_ACTIVE_INST_VMEM SQ_VALU_MFMA_BUSY_CYCLES SQ_LDS_BANK_CONFLICT GRBM_GUI_ACTIVE --output-format csv -d $out/c${i}a -o c -- python3 tools/row_profile.py run $i > $out/c${i}a.log 2>&1
  timeout -s KILL 90 rocprofv3 --pmc FETCH_SIZE --output-format csv -d $out/c${i}b -o c -- python3 tools/row_profile.py run $i > $out/c${i}b.log 2>&1
  timeout -s KILL 90 rocprofv3 --pmc WRITE_SIZE --output-format csv -d $out/c${i}c -o c -- python3 tools/row_profile.py run $i > $out/c${i}c.log 2>&1
  echo "counters of case $i taken"
done
