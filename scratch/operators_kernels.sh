#!/bin/bash
# rocprofv3 over every case of scratch/operators_kernels.py -> the file named (kept as profiles/operators/kernels.csv)
R=$(cd "$(dirname "$0")/.." && pwd)
OUT=$(realpath "${1:?file to write}")
cd /tmp && export TMPDIR=/tmp
echo "case,kernel,launches,median_us,min_us" > $OUT
python3 $R/scratch/operators_kernels.py names > /tmp/op_names 2>/dev/null || exit 1
while read -r c; do
  rm -rf /tmp/op_prof
  timeout -s KILL 90 rocprofv3 --kernel-trace --stats -d /tmp/op_prof -o c --output-format csv -- python3 $R/scratch/operators_kernels.py run "$c" > /tmp/op_prof.log 2>&1 < /dev/null \
    || { tail -3 /tmp/op_prof.log; exit 1; }
  python3 $R/scratch/operators_kernels.py table "$c" /tmp/op_prof | tee -a $OUT || exit 1
done < /tmp/op_names
