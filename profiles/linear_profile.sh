#!/bin/bash
# Times, kernel traces and counters of the linear layers on one box -> $1 (a folder): rates.txt, time.txt, trace.txt, counters.txt.
# usage (repo root): bash profiles/linear_profile.sh <folder> <built profiles/micro/linear_rates.hip>
set -e
R=$PWD; O=$R/$1; mkdir -p $O
timeout -k 10 100 $2 > $O/rates.txt
timeout -k 10 150 python3 -u profiles/linear_profile.py time 2> $O/time.err > $O/time.txt
cd /tmp; export TMPDIR=/tmp
timeout -s KILL 150 rocprofv3 --kernel-trace --output-format csv -d $O/t -o t -- python3 $R/profiles/linear_profile.py run > $O/run.log 2>&1
timeout -s KILL 100 rocprofv3 --kernel-trace --output-format csv -d $O/h -o h -- python3 $R/profiles/linear_profile.py heads > $O/heads.log 2>&1
python3 $R/profiles/linear_profile.py trace $(find $O/t -name t_kernel_trace.csv) > $O/trace.txt
echo "hash heads:" >> $O/trace.txt
python3 $R/profiles/linear_profile.py trace $(find $O/h -name h_kernel_trace.csv) >> $O/trace.txt
W="8192x8192x8192 16384-of-32 32-of-64 512-of-8-256 3001 16x4096x4096 777"
timeout -s KILL 120 rocprofv3 --pmc GRBM_GUI_ACTIVE SQ_VALU_MFMA_BUSY_CYCLES SQ_BUSY_CYCLES SQ_LDS_BANK_CONFLICT SQ_LDS_IDX_ACTIVE --output-format csv -d $O/c1 -o c -- python3 $R/profiles/linear_profile.py run $W > $O/c1.log 2>&1
timeout -s KILL 120 rocprofv3 --pmc FETCH_SIZE --output-format csv -d $O/c2 -o c -- python3 $R/profiles/linear_profile.py run $W > $O/c2.log 2>&1
python3 $R/profiles/linear_profile.py counters $(find $O/c1 $O/c2 -name c_counter_collection.csv) > $O/counters.txt
rm -rf $O/t $O/h $O/c1 $O/c2
