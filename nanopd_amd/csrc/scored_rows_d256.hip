// The rows kernel of the scored attention ops at padded head dim 256
// (scored_rows.h).
#include "scored_rows.h"

template void npd::scored::launch_rows<256>(const npd::scored::Args&, int32_t, hipStream_t);
