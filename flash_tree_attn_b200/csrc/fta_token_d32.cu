#define FTA_INST_D 32
#include "fta_token_stage1.inc"
